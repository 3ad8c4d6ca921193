"""What the MXFP4 matrix-vector product refuses, on the host."""
import pytest
import torch

from catccos_amd import _lib, ops


def test_host_tensors():
    x, w, s = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="expected a GPU tensor"):
        ops.mxfp4_gemv(x, w, s)


# a call that is whole; the addresses are never reached
WHOLE = dict(x=4096, ld_x=64, x_type=0, b=4096, ld_b=32, b_scale=4096, ld_bs=2, out=4096, ld_out=8, out_type=0, m=2, n=8, k=64, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(x=None), "null pointer"), (dict(b=None), "null pointer"), (dict(b_scale=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(x_type=3), "unknown type"), (dict(out_type=-1), "unknown type"), (dict(k=0), "multiple of 32"), (dict(k=48), "multiple of 32"),
    (dict(ld_x=63), "pitch"), (dict(ld_b=16), "pitch"), (dict(ld_bs=1), "pitch"), (dict(ld_out=7), "pitch"), (dict(b=4104), "16-byte"),
    (dict(ld_b=40), "16-byte"), (dict(x=4097), "aligned"), (dict(x=4098, x_type=2), "aligned"), (dict(out=4097), "aligned"),
    (dict(out=4098, out_type=2), "aligned"), (dict(m=1 << 21), "too many rows")])
def test_bad_arguments_are_refused_before_a_launch(change, message):
    lib = _lib.load()
    assert lib.cmx_mxfp4_gemv(*{**WHOLE, **change}.values()) == -1
    assert message.encode() in lib.cmx_last_error()


@pytest.mark.parametrize("change", [dict(m=0), dict(n=0), dict(m=0, x=None)])
def test_nothing_to_do_is_no_error(change):
    assert _lib.load().cmx_mxfp4_gemv(*{**WHOLE, **change}.values()) == 0


@pytest.mark.parametrize("change,message", [
    (dict(n=(1 << 26) + 16, ld_out=1 << 27), "too many rows of b"), (dict(n=0xFFFFFFF0, ld_out=0xFFFFFFFF), "too many rows of b"),
    (dict(k=1 << 30, ld_x=1 << 30, ld_b=1 << 29, ld_bs=1 << 25), "at most 2^29")])
def test_sizes_that_32_bits_of_a_launch_cannot_hold(change, message):
    test_bad_arguments_are_refused_before_a_launch(change, message)


def test_pitches_and_sizes_past_32_bits_are_refused_in_front():
    far = torch.empty_strided((2, 64), (1 << 32, 1), dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="2\\^32"):
        ops._pitch(far, 64)
    assert ops._pitch(far[:1], 64) == 64                              # (the stride of a single row says nothing)
    for call in (lambda: ops._fits(1 << 32), lambda: ops._fits(5 | -3), lambda: ops.mxfp4_moe_ffn_workspace_bytes(1 << 32, 64, 1),
                 lambda: ops.mxfp4_moe_ffn_workspace_bytes(1, 64, -1)):
        with pytest.raises(ValueError, match="2\\^32"):
            call()
    ops._fits((1 << 32) - 1)
