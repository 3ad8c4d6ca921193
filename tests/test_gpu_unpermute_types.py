"""The weighted way back and its gradients at the types that they share, and the ones that only the gradients take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(x):
    g = torch.Generator(device="cuda").manual_seed(11)
    tokens, top_k, h = 37, 3, 136
    to = torch.randperm(tokens * top_k, generator=torch.Generator().manual_seed(3)).int().cuda()
    y = torch.randn((tokens * top_k, h), generator=g, device="cuda").to(x)
    return y, to, torch.softmax(torch.randn((tokens, top_k), generator=g, device="cuda"), dim=1)


@pytest.mark.parametrize("x", [torch.float16, torch.float32])
def test_rows_that_are_not_bf16_are_refused(x):
    from catccos_amd import ops
    y, to, probs = _case(x)
    with pytest.raises(AssertionError):
        ops.moe_token_unpermute(y, to, probs)


def test_bf16_rows_as_numbers_and_as_bits():
    from catccos_amd import ops
    y, to, probs = _case(torch.bfloat16)
    got = ops.moe_token_unpermute(y, to, probs)
    want = (y.double()[to.long()].view(37, 3, 136) * probs.double()[:, :, None]).sum(dim=1)
    # three products and two additions in fp32, one rounding to 8 bits
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.001 + (y.double().abs()[to.long()].view(37, 3, 136) * probs.double()[:, :, None]).sum(dim=1) * 5 * 2.0 ** -24).all())
    for bits in (torch.int16, torch.uint16):
        assert torch.equal(ops.moe_token_unpermute(y.view(bits), to, probs).view(torch.bfloat16), got)
    wide = torch.full((y.shape[0], 152), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :136] = y
    assert torch.equal(ops.moe_token_unpermute(wide[:, :136], to.view(37, 3), probs), got)
