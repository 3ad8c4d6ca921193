"""What the way to the experts' order and the gradients of both ways refuse, on the host."""
import pytest
import torch

from catccos_amd import _lib, ops

PERMUTE = dict(x=4096, ld_x=8, to=4096, out=4096, ld_out=8, rows=4, tokens=2, hidden=8, top_k=2, element_bytes=2, zero_rest=0, stream=None)
PERMUTE_GRAD = dict(dy=4096, ld_dy=8, rows=4, to=4096, dx=4096, ld_dx=8, tokens=2, hidden=8, top_k=2, type=0, stream=None)
UNPERMUTE_GRAD = dict(dout=4096, ld_dout=8, y=4096, ld_y=8, rows=4, to=4096, probs=4096, dy=4096, ld_dy=8, dprobs=4096, tokens=2, hidden=8, top_k=2, type=0, zero_rest=0, stream=None)
CALLS = {"cmx_moe_token_permute": PERMUTE, "cmx_moe_token_permute_grad": PERMUTE_GRAD, "cmx_moe_token_unpermute_grad": UNPERMUTE_GRAD}


def test_host_tensors():
    x, to = torch.zeros(4, 8), torch.zeros(8, dtype=torch.int32)
    for call in (lambda: ops.moe_token_permute(x, to, 2), lambda: ops.moe_token_permute_grad(x, to, 2), lambda: ops.moe_token_unpermute_grad(x, x, to, torch.zeros(4, 2))):
        with pytest.raises(ValueError, match="expected a GPU tensor"):
            call()


ALL = [(dict(top_k=0), "top_k"), (dict(top_k=65), "top_k"), (dict(tokens=1 << 30), "2^31"), (dict(rows=1 << 31), "2^31"), (dict(to=None), "null pointer")]


@pytest.mark.parametrize("name,change,message", [(name, *a) for name in CALLS for a in ALL] + [
    ("cmx_moe_token_permute", *a) for a in ((dict(x=None), "null pointer"), (dict(out=None), "null pointer"), (dict(element_bytes=8), "1, 2 or 4"), (dict(ld_x=7), "pitch"), (dict(ld_out=7), "pitch"),
                                            (dict(x=4097), "aligned"), (dict(out=4098, element_bytes=4), "aligned"),
                                            (dict(tokens=1 << 29, hidden=1 << 20, ld_x=1 << 20, ld_out=1 << 20), "too many elements"))] + [
    ("cmx_moe_token_permute_grad", *a) for a in ((dict(dy=None), "null pointer"), (dict(dx=None), "null pointer"), (dict(type=3), "unknown type"), (dict(ld_dy=7), "pitch"), (dict(ld_dx=7), "pitch"),
                                                 (dict(dy=4097), "aligned"), (dict(dx=4098, type=2), "aligned"),
                                                 (dict(tokens=1 << 29, hidden=1 << 20, ld_dy=1 << 20, ld_dx=1 << 20), "too many elements"))] + [
    ("cmx_moe_token_unpermute_grad", *a) for a in ((dict(dout=None), "null pointer"), (dict(y=None), "null pointer"), (dict(probs=None), "null pointer"), (dict(dy=None), "null pointer"),
                                                   (dict(dprobs=None), "null pointer"), (dict(type=-1), "unknown type"), (dict(ld_dout=7), "pitch"), (dict(ld_y=7), "pitch"),
                                                   (dict(ld_dy=7), "pitch"), (dict(dout=4097), "aligned"), (dict(tokens=1 << 29), "too many tokens"))])
def test_refused_before_a_launch(name, change, message):
    lib = _lib.load()
    assert getattr(lib, name)(*{**CALLS[name], **change}.values()) == -1
    assert message.encode() in lib.cmx_last_error()


@pytest.mark.parametrize("name,change", [("cmx_moe_token_permute", dict(tokens=0)), ("cmx_moe_token_permute", dict(rows=0)), ("cmx_moe_token_permute", dict(hidden=0)),
                                         ("cmx_moe_token_permute_grad", dict(tokens=0)), ("cmx_moe_token_permute_grad", dict(hidden=0)), ("cmx_moe_token_unpermute_grad", dict(tokens=0))])
def test_nothing_to_do_is_no_error(name, change):
    assert getattr(_lib.load(), name)(*{**CALLS[name], **change}.values()) == 0
