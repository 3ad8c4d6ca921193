"""What the MXFP4 FFN refuses, on the host."""
import pytest
import torch

from catccos_amd import _lib, ops


def test_host_tensors():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    args = (torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2), u8(4, 128, 32), u8(4, 128, 2), u8(4, 64, 32),
            u8(4, 64, 2))
    with pytest.raises(ValueError, match="expected a GPU tensor"):
        ops.mxfp4_moe_ffn(*args)


# a call that is whole; the addresses are never reached
WHOLE = dict(x=4096, idx=4096, gate=4096, w1=4096, w1s=4096, w2=4096, w2s=4096, out=4096, workspace=4096, m=2, k=64, n=128, experts=4, top_k=2, stream=None)


@pytest.mark.parametrize("change,message", [(dict([(name, None)]), "null pointer") for name in list(WHOLE)[:9]] + [
    (dict(k=0), "k must"), (dict(k=48), "k must"), (dict(n=0), "n must"), (dict(n=96), "n must"), (dict(experts=0), "experts"), (dict(experts=1 << 31), "experts"),
    (dict(top_k=0), "top_k"), (dict(top_k=65), "top_k"), (dict(m=1 << 30, top_k=2), "too many tokens"), (dict(m=1 << 23), "too many tokens"),
    (dict(w1=4104), "16-byte"), (dict(w2=4104), "16-byte"), (dict(workspace=4224), "256-byte"), (dict(idx=4098), "aligned"), (dict(gate=4097), "aligned"),
    (dict(x=4104), "16-byte"), (dict(out=4097), "aligned")])
def test_bad_arguments_are_refused_before_a_launch(change, message):
    lib = _lib.load()
    assert lib.cmx_mxfp4_moe_ffn(*{**WHOLE, **change}.values()) == -1
    assert message.encode() in lib.cmx_last_error()


def test_no_tokens_and_the_workspace():
    lib = _lib.load()
    assert lib.cmx_mxfp4_moe_ffn(*{**WHOLE, "m": 0, "x": None}.values()) == 0
    need = ops.mxfp4_moe_ffn_workspace_bytes(32, 4096, 8)
    assert need >= 256 * 2048 * 4 and need % 256 == 0
    assert ops.mxfp4_moe_ffn_workspace_bytes(1 << 20, 4096, 8) >= (1 << 23) * 2048 * 4          # past 32 bits


@pytest.mark.parametrize("change,message", [(dict(k=(1 << 26) + 32), "at most 2^26"), (dict(n=(1 << 26) + 64), "at most 2^26"), (dict(n=0xFFFFFFC0), "at most 2^26")])
def test_sizes_that_32_bits_of_a_launch_cannot_hold(change, message):
    test_bad_arguments_are_refused_before_a_launch(change, message)
