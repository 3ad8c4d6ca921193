"""What the norm refuses, on the host."""
import pytest
import torch

from catccos_amd import _lib, ops


def test_host_tensors_and_other_devices(monkeypatch):
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm(x, w, residual=x), lambda: ops.rms_norm_quant(x, w)):
        with pytest.raises(ValueError, match="expected a GPU tensor"):
            call()

    class Elsewhere(torch.Tensor):
        def get_device(self):
            return 1
    monkeypatch.setattr(ops, "_device", lambda: 0)
    away = x.as_subclass(Elsewhere)
    with pytest.raises(ValueError, match=r"current device \(0\), not on device 1"):
        ops.rms_norm(away, w)
    monkeypatch.setattr(ops, "_device", lambda: 1)
    with pytest.raises(TypeError, match="expected a tensor"):
        ops.rms_norm(away, (torch.bfloat16, 64))


# a call that is whole: x, ld_x, residual, ld_residual, weight, total, ld_total, y, ld_y, codes, ld_codes, scales, ld_scales, rows, cols, eps, type,
# weight_type, fmt, stream; the addresses are never reached
WHOLE = dict(x=4096, ld_x=96, residual=4096, ld_residual=96, weight=4096, total=4096, ld_total=96, y=4096, ld_y=96, codes=4096, ld_codes=96, scales=4096,
             ld_scales=4, rows=2, cols=96, eps=0, type=0, weight_type=0, fmt=0, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(x=None), "null pointer"), (dict(weight=None), "null pointer"), (dict(y=None, codes=None, scales=None), "nothing to write"),
    (dict(scales=None), "come together"), (dict(codes=None), "come together"), (dict(residual=None), "total needs a residual"),
    (dict(ld_x=95), "pitch"), (dict(ld_residual=95), "pitch"), (dict(ld_total=95), "pitch"), (dict(ld_y=95), "pitch"), (dict(ld_codes=95), "pitch"),
    (dict(ld_scales=2), "pitch"), (dict(x=4097), "aligned"), (dict(y=4097), "aligned"), (dict(weight=4098, weight_type=2), "aligned"),
    (dict(type=3), "unknown type"), (dict(weight_type=1), "weight"), (dict(fmt=3), "unknown element format"),
    (dict(eps=ops._bits(-1e-6)), "eps"), (dict(eps=ops._bits(float("nan"))), "eps"), (dict(eps=ops._bits(float("inf"))), "eps"),
    (dict(cols=(1 << 30) + 1, ld_x=1 << 31, ld_residual=1 << 31, ld_total=1 << 31, ld_y=1 << 31, ld_codes=1 << 31, ld_scales=1 << 26), "too long")])
def test_bad_arguments_are_refused_before_a_launch(change, message):
    lib = _lib.load()
    assert lib.cmx_rms_norm_quant(*{**WHOLE, **change}.values()) == -1
    assert message.encode() in lib.cmx_last_error()


@pytest.mark.parametrize("change", [dict(rows=0), dict(cols=0), dict(rows=0, x=None, y=None)])
def test_nothing_to_do_is_no_error(change):
    assert _lib.load().cmx_rms_norm_quant(*{**WHOLE, **change}.values()) == 0


def test_eps_as_bits():
    assert ops._bits(1.0) == 0x3F800000 and ops._bits(0.0) == 0
    assert ops._bits(1e300) == 0x7F800000                         # (which the entry point refuses)


@pytest.mark.parametrize("rows,cols", [((1 << 26) + 1, 1), (0xFFFFFFFF, 1), (1 << 24, 1040), (1 << 22, 8200), (1 << 22, 20000)])
def test_more_rows_than_a_launch_has_threads_for(rows, cols):
    lib = _lib.load()
    pitch = 20000
    assert lib.cmx_rms_norm_quant(*{**WHOLE, "rows": rows, "cols": cols, **{name: pitch for name in WHOLE if name.startswith("ld_")}}.values()) == -1
    assert b"too many rows" in lib.cmx_last_error()
