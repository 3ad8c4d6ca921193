"""Token rows to the experts' order, and the gradients of both ways, against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CASES = [(1, 1, 1), (1, 8, 7168), (3, 2, 7), (45, 3, 1000), (777, 3, 1001), (300, 8, 64), (33, 64, 130), (4000, 6, 256), (5000, 1, 72)]


def _table(tokens, top_k, seed, dropped=0.0):
    """A permutation of the routes with some of them dropped."""
    g = torch.Generator().manual_seed(seed)
    to = torch.randperm(tokens * top_k, generator=g).int()
    if dropped:
        to[torch.rand(tokens * top_k, generator=g) < dropped] = -1
    return to.cuda()


def _rows(shape, x, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(DTYPES[x])


@pytest.mark.parametrize("tokens,top_k,h", CASES)
@pytest.mark.parametrize("dropped", [0.0, 0.4, 1.0])
def test_permute(tokens, top_k, h, dropped):
    from catccos_amd import ops
    to = _table(tokens, top_k, tokens + h, dropped)
    live = to >= 0
    for x in (_rows((tokens, h), "bf16", 1), _rows((tokens, h), "fp32", 2), torch.randint(0, 256, (tokens, h), dtype=torch.uint8, device="cuda")):
        want = torch.zeros((tokens * top_k, h), dtype=x.dtype, device="cuda")
        want[to[live].long()] = x.repeat_interleave(top_k, dim=0)[live]
        assert torch.equal(ops.moe_token_permute(x, to, top_k), want)
        # into more rows than there are routes, and fewer: what no route is sent to stays
        kept = torch.full((tokens * top_k + 5, h + 3), 9, dtype=x.dtype, device="cuda")
        out = kept[:, 1:h + 1]
        ops.moe_token_permute(x, to, top_k, out=out)
        hit = torch.zeros(tokens * top_k + 5, dtype=torch.bool, device="cuda")
        hit[to[live].long()] = True
        assert torch.equal(out[:-5][hit[:-5]], want[hit[:-5]]) and bool((out[~hit] == 9).all()) and bool((kept[:, h + 1:] == 9).all()) and bool((kept[:, 0] == 9).all())
        few = torch.full((tokens * top_k // 2, h), 9, dtype=x.dtype, device="cuda")
        ops.moe_token_permute(x, to, top_k, out=few)
        n = few.shape[0]
        assert torch.equal(few[hit[:n]], want[:n][hit[:n]]) and bool((few[~hit[:n]] == 9).all())


@pytest.mark.parametrize("tokens,top_k,h", CASES)
@pytest.mark.parametrize("x", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dropped", [0.0, 0.4])
def test_gradients(tokens, top_k, h, x, dropped):
    from catccos_amd import ops
    to = _table(tokens, top_k, tokens + h, dropped)
    y, dout = _rows((tokens * top_k, h), x, 3), _rows((tokens, h), x, 4)
    probs = torch.softmax(_rows((tokens, top_k), "fp32", 5), dim=1)
    live = (to >= 0).view(tokens, top_k)
    at = to.long().clamp_min(0).view(tokens, top_k)
    rows = y.double()[at] * live[:, :, None]
    half = torch.finfo(DTYPES[x]).eps / 2
    # top_k - 1 additions in fp32, one rounding
    dx = ops.moe_token_permute_grad(y, to, top_k)
    want = rows.sum(dim=1)
    bound = want.abs() * (half if x != "fp32" else 0) * 1.001 + rows.abs().sum(dim=1) * top_k * 2.0 ** -24 + 6e-8 * (x == "fp16")
    assert dx.dtype == y.dtype and bool(((dx.double() - want).abs() <= bound).all())
    dy, dprobs = ops.moe_token_unpermute_grad(dout, y, to, probs)
    want = torch.zeros((tokens * top_k, h), dtype=torch.float64, device="cuda")
    want[at[live]] = (probs.double()[:, :, None] * dout.double()[:, None, :])[live]
    # a product in fp32, one rounding
    assert bool(((dy.double() - want).abs() <= want.abs() * (half * 1.001 + 2.0 ** -24) + 6e-8 * (x == "fp16")).all())
    each = dout.double()[:, None, :] * rows
    # a multiply-add for each of a thread's elements, 6 additions in a wavefront, 4 across
    n = -(-h // 256) + 16
    assert bool(((dprobs.double() - each.sum(dim=2)).abs() <= each.abs().sum(dim=2) * n * 2.0 ** -24).all())
    assert bool((dprobs[~live] == 0).all())


def test_the_gradients_are_those_of_differences():
    """Of L = sum(unpermute(y, probs) * w) and L = sum(permute(x) * w), which are linear in every input: a difference over a whole step is the gradient."""
    from catccos_amd import ops
    tokens, top_k, h = 6, 3, 40
    to = _table(tokens, top_k, 2)
    g = torch.Generator(device="cuda").manual_seed(1)
    whole = lambda *shape: torch.randint(-3, 4, shape, generator=g, device="cuda").float()     # small whole numbers: every sum is exact
    y, probs, w = whole(tokens * top_k, h), whole(tokens, top_k), whole(tokens, h)
    combine = lambda y, p: float((ops.moe_token_unpermute(y.to(torch.bfloat16), to, p).float() * w).sum())
    dy, dprobs = ops.moe_token_unpermute_grad(w, y, to, probs)
    base = combine(y, probs)
    for r, c in ((0, 0), (5, 39), (17, 20)):
        moved = y.clone()
        moved[r, c] += 1
        assert combine(moved, probs) - base == float(dy[r, c])
    for t, r in ((0, 0), (5, 2), (3, 1)):
        moved = probs.clone()
        moved[t, r] += 1
        assert combine(y, moved) - base == float(dprobs[t, r])
    x, v = whole(tokens, h), whole(tokens * top_k, h)
    spread = lambda x: float((ops.moe_token_permute(x, to, top_k) * v).sum())
    dx = ops.moe_token_permute_grad(v, to, top_k)
    for t, c in ((0, 0), (5, 39), (2, 7)):
        moved = x.clone()
        moved[t, c] += 1
        assert spread(moved) - spread(x) == float(dx[t, c])


def test_dropped_routes_of_not_finite_rows_add_nothing():
    from catccos_amd import ops
    to = torch.tensor([0, -1, 7, 1], dtype=torch.int32, device="cuda")          # (7 is behind the rows)
    y = torch.ones((2, 16), device="cuda")
    dout = torch.full((2, 16), float("inf"), device="cuda")
    dout[0] = 1
    probs = torch.ones((2, 2), device="cuda")
    dy, dprobs = ops.moe_token_unpermute_grad(dout, y, to, probs)
    assert dprobs[0].tolist() == [16.0, 0.0] and dprobs[1, 0] == 0 and bool((dy[0] == 1).all()) and bool(torch.isinf(dy[1]).all())
    assert bool((ops.moe_token_permute_grad(y, to, 2) == 1).all())


def test_rows_past_4_gib():
    from catccos_amd import ops
    h, rows = 65536, 70000
    y = torch.zeros((rows, h), dtype=torch.uint8, device="cuda")
    x = torch.arange(4, dtype=torch.uint8, device="cuda")[:, None].expand(4, h).contiguous() + 1
    to = torch.tensor([69999, 66000, 0, -1], dtype=torch.int32, device="cuda")
    ops.moe_token_permute(x, to, 1, out=y)
    assert bool((y[69999] == 1).all()) and bool((y[66000] == 2).all()) and bool((y[0] == 3).all()) and not bool(y[1:66000:997].any()) and not bool(y[69998].any())
    half = y.view(torch.bfloat16)
    dx = ops.moe_token_permute_grad(half, to, 1)
    assert torch.equal(dx[0], half[69999]) and torch.equal(dx[1], half[66000]) and not bool(dx[3].any())
