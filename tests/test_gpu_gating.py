"""The gate against the definition in 64 bits: the same indices, and weights to what fp32 leaves of them."""
import math

import pytest
import torch

from catccos_amd import ops

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Relative error of a weight in fp32.  Softmax: |z - max| * 2^-24 from the difference (|z| stays below 10 here, so at most 20), exp 2 units, 16 + 6
# additions, and the same for the sum that divides it, a division and the scale: (20 + 2 + 22 + 2) * 2 * 2^-24 < 2^-17
WEIGHT_LOSS = 2.0 ** -17


def _definition(z, top_k, score, bias, groups, top_groups, group_best, renormalize, scale):
    z = z.double()
    if score == "softmax":
        most = z.amax(dim=1, keepdim=True)
        s = torch.where(z == -math.inf, 0.0, torch.exp(z - most))
        total = s.sum(dim=1, keepdim=True)
        s = torch.where(total == 0, 0.0, s / total)
    else:
        s = 1 / (1 + torch.exp(-z))
    c = s if bias is None else s + bias.double()
    t, e = z.shape
    if groups > 1:
        c = c.view(t, groups, -1)
        best = c.sort(dim=2, descending=True).values[:, :, :group_best].sum(dim=2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        closed = torch.ones_like(best, dtype=torch.bool).scatter(1, kept, False)
        order = torch.where(closed[:, :, None].expand_as(c), 1, 0).reshape(t, e)
        c = c.reshape(t, e)
        by_value = c.sort(dim=1, descending=True, stable=True).indices
        idx = by_value.gather(1, order.gather(1, by_value).sort(dim=1, stable=True).indices)[:, :top_k]      # closed groups behind the open ones
    else:
        idx = c.sort(dim=1, descending=True, stable=True).indices[:, :top_k]
    w = s.gather(1, idx)
    if renormalize:
        total = w.sum(dim=1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
    return idx, w * scale


def _check(z, top_k, score="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    idx, w = ops.moe_gating(z, top_k, score, bias, groups, top_groups, group_best, renormalize, scale)
    want_idx, want_w = _definition(z, top_k, score, bias, groups, top_groups, group_best, renormalize, scale)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and idx.shape == w.shape == (z.shape[0], top_k)
    rows = (idx.long() != want_idx).any(dim=1).nonzero().flatten().tolist()
    assert not rows, f"{len(rows)} rows differ, the first: {rows[0]}: {idx[rows[0]].tolist()} for {want_idx[rows[0]].tolist()}"
    err = (w.double() - want_w).abs()
    assert bool((err <= want_w.abs() * WEIGHT_LOSS + 2.0 ** -140).all()), float((err / want_w.abs().clamp_min(1e-300)).max())


def _logits(tokens, experts, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (std * torch.randn((tokens, experts), generator=g, device="cuda")).to(DTYPES[dtype]), 0.05 * torch.randn(experts, generator=g, device="cuda")


SIZES = [(1, 1), (2, 2), (8, 1), (8, 8), (16, 4), (17, 3), (32, 32), (33, 5), (64, 6), (100, 10), (128, 64), (160, 7), (255, 9), (256, 8), (257, 8), (384, 64),
         (512, 16), (1000, 12), (1024, 64)]


@pytest.mark.parametrize("experts,top_k", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_every_size(experts, top_k, dtype):
    for tokens in (1, 5, 67, 2051):
        z, bias = _logits(tokens, experts, dtype, experts + tokens)
        for score in ("softmax", "sigmoid"):
            for b in (None, bias):
                _check(z, top_k, score, b, renormalize=tokens != 67, scale=2.5 if tokens == 5 else 1.0)


@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(8, 2, 1, 4), (8, 8, 3, 3), (16, 4, 2, 5), (24, 3, 2, 9), (60, 20, 7, 6), (64, 64, 10, 10), (256, 8, 4, 8),
                                                              (256, 16, 3, 30), (320, 64, 9, 33), (512, 32, 32, 64), (1000, 10, 2, 8), (1024, 16, 5, 64)])
@pytest.mark.parametrize("group_best", [1, 2])
def test_groups(experts, groups, top_groups, top_k, group_best):
    for tokens, dtype in ((1, "fp32"), (7, "bf16"), (2100, "fp32"), (2100, "bf16")):
        z, bias = _logits(tokens, experts, dtype, experts + tokens + group_best)
        for score in ("softmax", "sigmoid"):
            for b in (None, bias):
                _check(z, top_k, score, b, groups, top_groups, group_best, renormalize=tokens != 7)


@pytest.mark.parametrize("tokens", [3, 3000])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_index(tokens, score):
    for levels in (1, 2, 5):                                           # few different values: nearly everything ties
        g = torch.Generator(device="cuda").manual_seed(levels)
        z = torch.randint(0, levels, (tokens, 256), generator=g, device="cuda").float()
        for bias in (None, torch.zeros(256, device="cuda"), torch.randint(0, 2, (256,), generator=g, device="cuda").float()):
            _check(z, 8, score, bias)
            _check(z, 8, score, bias, 8, 4, 2)
            _check(z, 8, score, bias, 8, 4, 1)


@pytest.mark.parametrize("tokens", [16, 4096])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_values_that_fp32_cannot_tell_apart(tokens, score):
    """Logits that differ in their last bit only, and biases that make up for differences in the score to about the last bit of fp32: the order is still
    that of 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(11)
    base = torch.randn((tokens, 1), generator=g, device="cuda")
    step = torch.randint(-3, 4, (tokens, 256), generator=g, device="cuda", dtype=torch.int32)
    z = (base.expand(tokens, 256).contiguous().view(torch.int32) + step).view(torch.float32)
    _check(z, 8, score)
    _check(z, 8, score, torch.zeros(256, device="cuda"))
    _check(z, 8, score, torch.zeros(256, device="cuda"), 8, 4, 2)
    z = torch.randn((1, 256), generator=g, device="cuda").expand(tokens, 256).contiguous()
    s = torch.softmax(z[:1].double(), dim=1) if score == "softmax" else torch.sigmoid(z[:1].double())
    _check(z, 8, score, (0.75 - s[0]).float())
    _check(z, 8, score, (0.75 - s[0]).float(), 16, 4, 2)
    _check(z * 30, 8, score, torch.zeros(256, device="cuda"))           # sigmoids that fp32 rounds to one, exps that it loses


def test_masked_experts_and_rows_without_any():
    tokens, experts = 2500, 96
    z, bias = _logits(tokens, experts, "fp32", 4)
    z[:, 10:] = torch.where(torch.rand((tokens, experts - 10), device="cuda") < 0.9, -math.inf, z[:, 10:])
    z[7] = -math.inf
    z[8, 1:] = -math.inf
    z[9] = torch.finfo(torch.float32).min
    for score in ("softmax", "sigmoid"):
        for b in (None, bias, torch.where(torch.arange(experts, device="cuda") % 3 == 0, -math.inf, bias)):
            for part in (z, z[5:12]):
                _check(part, 16, score, b)
                _check(part, 16, score, b, 8, 4, 1)
    w = ops.moe_gating(z[7:8], 4)[1]
    assert bool((w == 0).all())


@pytest.mark.parametrize("tokens", [40, 2500])
def test_indices_stay_distinct_and_in_range_whatever_a_row_holds(tokens):
    g = torch.Generator(device="cuda").manual_seed(8)
    z = torch.randn((tokens, 256), generator=g, device="cuda")
    z = torch.where(torch.rand(z.shape, generator=g, device="cuda") < 0.6, math.nan, z)
    z = torch.where(torch.rand(z.shape, generator=g, device="cuda") < 0.1, math.inf, z)
    z[3] = math.nan
    z[4] = math.inf
    for score in ("softmax", "sigmoid"):
        for b in (None, torch.where(torch.arange(256, device="cuda") < 100, math.nan, 0.1), torch.full((256,), math.inf, device="cuda")):
            for args in ((1, 1, 1), (8, 4, 2), (8, 2, 1)):
                idx, w = ops.moe_gating(z, 32, score, b, *args)
                s = idx.long().sort(dim=1).values
                assert bool((s[:, 0] >= 0).all()) and bool((s[:, -1] < 256).all()) and bool((s[:, 1:] > s[:, :-1]).all())
                if score == "softmax":
                    assert bool(w.isnan().all())                        # every row here holds a NaN or +Inf
    # a NaN ranks behind the others
    z = torch.zeros((tokens, 64), device="cuda")
    z[:, ::2] = math.nan
    idx, _ = ops.moe_gating(z, 40, "sigmoid")
    assert bool((idx[:, :32] == torch.arange(1, 64, 2, device="cuda")).all()) and bool((idx[:, 32:] == torch.arange(0, 16, 2, device="cuda")).all())


def test_strided_rows_past_32_bits_and_no_rows():
    z, bias = _logits(9, 300, "bf16", 3)
    view = z[::2, 7:263]
    assert all(torch.equal(p, q) for p, q in zip(ops.moe_gating(view, 8), ops.moe_gating(view.contiguous(), 8)))
    apart = (1 << 32) - 8
    buf = torch.empty(apart + 256, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((2, 256), (apart, 1))
    far.copy_(z[:2, :256])
    assert all(torch.equal(p, q) for p, q in zip(ops.moe_gating(far, 8, "sigmoid", bias[:256], 8, 4, 2), ops.moe_gating(z[:2, :256], 8, "sigmoid", bias[:256], 8, 4, 2)))
    idx, w = ops.moe_gating(z[:0], 8)
    assert idx.shape == w.shape == (0, 8)


def test_on_a_side_stream_and_captured():
    ops.init()
    z, bias = _logits(2100, 256, "fp32", 6)
    call = lambda: ops.moe_gating(z, 8, "sigmoid", bias, 8, 4, 2, scale=2.5)
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for rep in range(3):
        z.copy_(torch.randn(z.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, call())), rep


def test_into_the_routing_sort():
    """The gate's answer is what moe_init_routing takes."""
    z, _ = _logits(777, 256, "bf16", 2)
    idx, w = ops.moe_gating(z, 8)
    order, place, counts = ops.moe_init_routing(idx, 256)
    assert torch.equal(counts.long(), torch.bincount(idx.flatten().long(), minlength=256))
    assert torch.equal(order.long(), idx.flatten().long().sort(stable=True).indices)
    assert bool(((w.sum(dim=1) - 1).abs() < 1e-5).all())


@pytest.mark.parametrize("tokens", [37, 3700])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(434, 2, 1, 4), (272, 4, 4, 1), (230, 2, 2, 11), (500, 10, 3, 8), (66, 33, 9, 16), (448, 64, 20, 8), (1000, 5, 2, 9),
                                                              (512, 1, 1, 8), (512, 8, 4, 16), (32, 2, 1, 16), (45, 15, 7, 3)])
def test_groups_of_every_size_and_many_experts(tokens, experts, groups, top_groups, top_k):
    """Groups that do not fall on whole lanes, more of them than a row has lanes, more experts than a row has by the lane; few rows and many."""
    g = torch.Generator(device="cuda").manual_seed(experts + tokens)
    for dtype, score, group_best in ((torch.float32, "softmax", 1), (torch.float16, "sigmoid", 2), (torch.bfloat16, "softmax", 2)):
        z = torch.randn((tokens, experts), generator=g, device="cuda").to(dtype)
        for bias in (None, 0.1 * torch.randn(experts, generator=g, device="cuda")):
            _check(z, top_k, score, bias, groups, top_groups, group_best)


@pytest.mark.parametrize("tokens", [40, 4000])
@pytest.mark.parametrize("top_k", [2, 15, 16, 17, 24, 40, 64])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_pairs_that_fp32_cannot_tell_apart(tokens, top_k, score):
    """Scores in pairs: 2^-24 of a logit inside a pair, 1/16 between pairs, in random order; chosen whole pairs, a pair in part, and with a bias that swaps
    some; short rows that are taken whole; and rows whose scores all lie together."""
    g = torch.Generator(device="cuda").manual_seed(top_k)
    experts = 96
    level = -torch.arange(experts // 2, device="cuda").repeat_interleave(2) / 16.0 - 0.5
    z = torch.where(torch.arange(experts, device="cuda") % 2 == 1, torch.nextafter(level, torch.zeros_like(level)), level)
    z = z[torch.rand((tokens, experts), generator=g, device="cuda").argsort(dim=1)]
    bias = torch.where(torch.rand(experts, generator=g, device="cuda") < 0.5, 2.0 ** -26, -2.0 ** -27)
    for b in (bias, None):
        _check(z, top_k, score, b)
        _check(z[:, :64], top_k, score, None if b is None else b[:64], 4, 4, 2)
    _check(z[:, :top_k], top_k, score, bias[:top_k].contiguous())
    _check(1e-6 * torch.randn((tokens, experts), generator=g, device="cuda"), top_k, score, bias)


@pytest.mark.parametrize("tokens", [300, 4000])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_of_different_size_under_cancelling_biases(tokens, score):
    """Small scores, which fp32 knows to many places, and large ones, brought together by biases: two small ones that are clear of each other settle nothing
    about a large one that fp32 puts behind both."""
    g = torch.Generator(device="cuda").manual_seed(21)
    experts = 64
    large = torch.arange(experts, device="cuda") % 2 == 1
    base = torch.where(large, 1 + 3 * torch.rand(experts, generator=g, device="cuda"), -7 + 2 * torch.rand(experts, generator=g, device="cuda"))
    s = torch.softmax(base.double(), dim=0) if score == "softmax" else torch.sigmoid(base.double())
    apart = (2 * torch.rand(experts, generator=g, device="cuda").double() - 1) * (5e-8 if score == "softmax" else 4e-7)
    bias = ((0.0005 if score == "softmax" else 0.01) + apart - s).float()
    step = torch.randint(-3, 4, (tokens, experts), generator=g, device="cuda", dtype=torch.int32)
    z = (base.expand(tokens, experts).contiguous().view(torch.int32) + step).view(torch.float32)
    for top_k in (1, 2, 5, 16, 30):
        _check(z, top_k, score, bias)
        _check(z, min(top_k, 8), score, bias, 4, 1, 1)
        _check(z, top_k, score, bias, 4, 2, 2)


def test_a_large_score_behind_two_small_ones_that_are_clear():
    for z, bias in (([-60.0, -60.0, 2.0], [1.49e-7, 1.34e-7, 1.69e-7 - 1 / (1 + math.exp(-2.0))]), ([-7.0, -7.0, 2.4627566], [0.009088952, 0.00908894, -0.91148925])):
        for tokens in (1, 4000):
            row = torch.tensor(z, device="cuda").expand(tokens, 3).contiguous()
            for top_k in (1, 2, 3):
                _check(row, top_k, "sigmoid", torch.tensor(bias, device="cuda"))


@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(512, 64, 64, 64), (320, 64, 40, 64), (384, 64, 13, 58), (520, 52, 30, 64), (512, 64, 8, 64)])
def test_the_most_groups_and_the_largest_top_k_of_many_rows(experts, groups, top_groups, top_k):
    """Workgroups that hold more than 64 KiB of lists: up to 512 experts, 14 rows and more to a CU."""
    tokens = 14 * torch.cuda.get_device_properties(0).multi_processor_count + 5
    z, bias = _logits(tokens, experts, "fp32", experts)
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            _check(z, top_k, score, b, groups, top_groups, 2)
    _check(z.half(), top_k, "sigmoid", bias, groups, top_groups, 1)


def test_the_largest_workgroups_captured_right_after_init():
    """Their first launch inside a stream capture, after cmx_init() alone (tests/capture_gating_child.py)."""
    import os
    import subprocess
    import sys
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "capture_gating_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "CAPTURE-OK" in r.stdout, (r.returncode, r.stdout[-2000:], r.stderr[-2000:])


@pytest.mark.parametrize("tokens", [41, 4001])
def test_softmax_rows_that_hold_a_nan_or_inf_have_no_order(tokens):
    """Every score is NaN, which counts as -Inf: the lowest indices, whatever else the row holds, where scores are compared; the rows beside are not touched."""
    g = torch.Generator(device="cuda").manual_seed(31)
    z = torch.randn((tokens, 96), generator=g, device="cuda")
    z = torch.where(torch.rand(z.shape, generator=g, device="cuda") < 0.5, -math.inf, z)
    poisoned = torch.arange(tokens, device="cuda") % 3 != 0
    z[poisoned, 70] = torch.where(torch.arange(tokens, device="cuda") % 2 == 0, math.nan, math.inf)[poisoned]
    bias = 0.5 + 0.1 * torch.randn(96, generator=g, device="cuda")
    for b, args in ((bias, (1, 1, 1)), (bias, (8, 4, 2)), (bias, (8, 3, 1)), (bias, (48, 20, 2)), (None, (8, 4, 2)), (None, (48, 20, 2))):
        for top_k in (1, 5, 20, 36):
            idx, w = ops.moe_gating(z, top_k, "softmax", b, *args)
            assert bool((idx[poisoned] == torch.arange(top_k, device="cuda")).all()), (args, top_k)
            assert bool(w[poisoned].isnan().all())
            _check(z[~poisoned], top_k, "softmax", b, *args)
            want = ops.moe_gating(z[~poisoned], top_k, "softmax", b, *args)
            assert torch.equal(idx[~poisoned], want[0])


@pytest.mark.parametrize("tokens", [37, 4003])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_without_a_bias_the_order_is_the_logits_where_scores_are_lost(tokens, score):
    """Logits whose scores even 64 bits round to one or to zero, in groups that are compared by sums of two scores: the kept groups' experts come in the order
    of their logits, and masked ones behind all others."""
    g = torch.Generator(device="cuda").manual_seed(41)
    z = torch.randn((tokens, 64), generator=g, device="cuda")
    z = torch.where(torch.rand(z.shape, generator=g, device="cuda") < 0.3, -math.inf, z * 30 - 2000)      # scores of zero
    if score == "sigmoid":
        z[:, 5::9] = 60 + 10 * torch.rand((tokens, len(range(5, 64, 9))), generator=g, device="cuda")     # and of one
    else:
        z[:, 9] = 1.0
    for top_k in (1, 6, 14, 32):
        for kept in (8, 4):
            part = z
            if kept == 4:                                              # groups 1, 3, 5 and 7 stand out
                part = z.clone()
                for n in (1, 3, 5, 7):
                    part[:, 8 * n + 2], part[:, 8 * n + 3] = 3.0 + n, 2.0 + n
            idx, _ = ops.moe_gating(part, top_k, score, None, 8, kept, 2)
            key = torch.where(part == -math.inf, -1e30, part)          # masked ones last, but in front of those of closed groups
            if kept == 4:
                key = torch.where(torch.arange(64, device="cuda") // 8 % 2 == 1, key, -math.inf)
            assert torch.equal(idx.long(), key.sort(dim=1, descending=True, stable=True).indices[:, :top_k]), (top_k, kept)


@pytest.mark.parametrize("tokens", [3, 4001])
def test_a_logit_of_minus_inf_is_a_score_of_zero_and_a_bias_of_minus_inf_a_mask(tokens):
    z, _ = _logits(tokens, 64, "fp32", 51)
    masked = torch.arange(64, device="cuda") % 2 == 0
    for score in ("softmax", "sigmoid"):
        for args in ((1, 1, 1), (8, 8, 2), (8, 6, 1)):
            # -Inf in the logits: behind all others without a bias; with one, c is the bias
            away = torch.where(masked, -math.inf, z)
            idx, w = ops.moe_gating(away, 24, score, None, *args)
            assert not bool(masked[idx.long()].any()) and bool((w > 0).all())
            idx, w = ops.moe_gating(away, 24, score, torch.where(masked, 2.0, 0.0), *args)
            assert bool(masked[idx.long()].all()) and bool((w == 0).all())
            # in the bias: behind all others, whatever the logits
            idx, w = ops.moe_gating(torch.where(masked, z + 20, z), 24, score, torch.where(masked, -math.inf, 0.1), *args)
            assert not bool(masked[idx.long()].any()) and bool((w > 0).all())


@pytest.mark.parametrize("tokens", [5, 4001])
def test_weights_of_scores_that_fp32_cannot_hold(tokens):
    """Chosen scores below what fp32 holds: their quotients are not.  A weight is then a quotient of exponentials of differences between chosen logits, below
    10 here, and of their sum: fewer roundings than WEIGHT_LOSS counts."""
    g = torch.Generator(device="cuda").manual_seed(61)
    z = torch.randn((tokens, 64), generator=g, device="cuda")
    low = torch.where(torch.arange(64, device="cuda") % 4 == 0, 0.0, -math.inf)           # the bias keeps these 16 out of 64
    zero = torch.zeros(64, device="cuda")
    for shift in (30.0, 80.0, 95.0, 110.0, 400.0, 700.0):
        _check(z - shift, 8, "sigmoid", None)
        _check(z - shift, 8, "sigmoid", zero, 8, 4, 2)
        _check(z - shift, 16, "sigmoid", low, scale=2.5)
        far = torch.where(low == 0, z - shift, z)
        for args in ((1, 1, 1), (4, 4, 2)):
            _check(far, 16, "softmax", low, *args)
    # all alike: 1 / 8 each
    w = ops.moe_gating(torch.full((tokens, 64), -95.0, device="cuda"), 8, "sigmoid")[1]
    assert bool(((w - 0.125).abs() <= 2.0 ** -24).all())
    # not renormalised: the score itself, rounded where fp32 has fewer bits for it
    z = -80 - 20 * torch.rand((tokens, 64), generator=g, device="cuda")
    idx, w = ops.moe_gating(z, 8, "sigmoid", renormalize=False)
    want = torch.sigmoid(z.double()).gather(1, idx.long())
    assert bool(((w.double() - want).abs() <= want * WEIGHT_LOSS + 2.0 ** -148).all())
