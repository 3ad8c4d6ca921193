"""What the gate refuses, on the host."""
import pytest
import torch

from catccos_amd import _lib, ops


def test_host_tensors_and_other_devices(monkeypatch):
    z = torch.zeros(2, 64)
    for call in (lambda: ops.moe_gating(z, 4), lambda: ops.moe_gating(z, 4, bias=torch.zeros(64))):
        with pytest.raises(ValueError, match="expected a GPU tensor"):
            call()

    class Elsewhere(torch.Tensor):
        def get_device(self):
            return 3
    monkeypatch.setattr(ops, "_device", lambda: 0)
    with pytest.raises(ValueError, match="not on device 3"):
        ops.moe_gating(z.as_subclass(Elsewhere), 4)
    with pytest.raises(TypeError):
        ops.moe_gating(z, torch.tensor(2.5))                       # a whole number is asked for, not a tensor's address


# a call that is whole; the addresses are never reached
WHOLE = dict(logits=4096, ld=64, type=2, bias=4096, tokens=3, experts=64, top_k=4, score=1, groups=8, top_groups=4, group_best=2, renormalize=1,
             scale=ops._bits(2.5), idx=4096, weight=4096, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(logits=None), "null pointer"), (dict(idx=None), "null pointer"), (dict(weight=None), "null pointer"), (dict(ld=63), "pitch"),
    (dict(type=3), "unknown type"), (dict(type=-1), "unknown type"), (dict(score=2), "unknown score"), (dict(experts=0), "experts"),
    (dict(experts=1032, ld=2000), "experts"), (dict(groups=0), "groups"), (dict(groups=7), "groups"), (dict(groups=128, experts=128, ld=128), "groups"),
    (dict(top_groups=0), "top_groups"), (dict(top_groups=9), "top_groups"), (dict(group_best=0), "group_best"), (dict(group_best=3), "group_best"),
    (dict(top_k=0), "top_k"), (dict(top_k=33), "top_k"), (dict(top_k=65, experts=1024, ld=1024), "top_k"), (dict(tokens=1 << 30), "routes"),
    (dict(scale=ops._bits(float("inf"))), "scale"), (dict(scale=ops._bits(float("nan"))), "scale"), (dict(logits=4098), "aligned"),
    (dict(logits=4097, type=0), "aligned"), (dict(bias=4098), "aligned"), (dict(idx=4098), "aligned"), (dict(weight=4097), "aligned")])
def test_bad_arguments_are_refused_before_a_launch(change, message):
    lib = _lib.load()
    assert lib.cmx_moe_gating(*{**WHOLE, **change}.values()) == -1
    assert message.encode() in lib.cmx_last_error()


def test_nothing_to_do_is_no_error():
    assert _lib.load().cmx_moe_gating(*{**WHOLE, "tokens": 0, "logits": None}.values()) == 0


@pytest.mark.parametrize("tokens", [1 << 26, (1 << 31) - 1])
def test_more_tokens_than_a_launch_has_threads_for(tokens):
    lib = _lib.load()
    assert lib.cmx_moe_gating(*{**WHOLE, "tokens": tokens, "top_k": 1}.values()) == -1
    assert b"below 2^26" in lib.cmx_last_error()
