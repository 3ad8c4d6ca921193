"""What the FP8 quantiser and products with a scale for each block of 128 refuse, on the host."""
import pytest
import torch

from catccos_amd import _lib, ops


def test_host_tensors():
    x, u, s = torch.zeros(4, 128), torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 1)
    for call in (lambda: ops.fp8_block_quant(x), lambda: ops.fp8_block_gemm(u, s, u, s), lambda: ops.fp8_block_gmm(u, s, u[None], s[None, :1], torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="expected a GPU tensor"):
            call()
    with pytest.raises(ValueError, match="E4M3 or E5M2"):
        ops.fp8_block_quant(x, "E2M1")


# calls that are whole; the addresses are never reached
QUANT = dict(x=4096, ld_x=300, x_step=0, type=0, codes=4096, ld_codes=304, scales=4096, ld_scales=3, batch=1, rows=5, cols=300, fmt=0, square=0, transposed=0, pow2=0, stream=None)
GEMM = dict(a=4096, lda=256, a_scale=4096, ld_as=2, b=4096, ldb=256, b_scale=4096, ld_bs=2, b_rows=128, c=4096, ldc=8, m=2, n=8, k=256, fmt=0, out_type=0, workspace=None, stream=None)
GMM = dict(a=4096, lda=256, a_scale=4096, ld_as=2, b=4096, b_scale=4096, c=4096, ldc=8, sizes=4096, groups=3, m=2, n=8, k=256, fmt=0, out_type=0, zero_rest=0, stream=None)


def _refused(name, call, message):
    lib = _lib.load()
    assert getattr(lib, name)(*call.values()) == -1
    assert message.encode() in lib.cmx_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(x=None), "null pointer"), (dict(codes=None), "null pointer"), (dict(scales=None), "null pointer"), (dict(type=3), "unknown type"), (dict(fmt=2), "8-bit formats"),
    (dict(fmt=-1), "8-bit formats"), (dict(ld_x=299), "pitch"), (dict(ld_codes=303), "pitch"), (dict(ld_scales=2), "pitch"), (dict(x=4097), "aligned to their"),
    (dict(x=4098, type=2), "aligned to their"), (dict(scales=4098), "aligned to their"), (dict(codes=4104), "16-byte"), (dict(ld_codes=312), "16-byte"),
    (dict(batch=65536), "matrices"), (dict(rows=1 << 31), "at most 2^31"), (dict(transposed=1, ld_codes=0), "pitch"),
    (dict(rows=(1 << 31) - 1, cols=1 << 16, ld_x=1 << 16, ld_codes=1 << 16, ld_scales=1 << 9), "too many elements"),
    (dict(rows=(1 << 23) + (1 << 20), square=1), "too many rows")])
def test_quant_refuses_before_a_launch(change, message):
    _refused("cmx_fp8_block_quant", {**QUANT, **change}, message)


PRODUCT = [(dict(a=None), "null pointer"), (dict(a_scale=None), "null pointer"), (dict(b=None), "null pointer"), (dict(b_scale=None), "null pointer"), (dict(c=None), "null pointer"),
           (dict(fmt=2), "8-bit formats"), (dict(out_type=3), "unknown type"), (dict(k=0), "multiple of 16"), (dict(k=200), "multiple of 16"), (dict(lda=240), "pitch"),
           (dict(ld_as=1), "pitch"), (dict(ldc=7), "pitch"), (dict(a=4104), "16-byte"), (dict(b=4104), "16-byte"), (dict(lda=264), "16-byte"), (dict(a_scale=4098), "aligned to their"),
           (dict(b_scale=4097), "aligned to their"), (dict(c=4097), "aligned to their"), (dict(c=4098, out_type=2), "aligned to their"), (dict(m=1 << 31), "at most 2^31"),
           (dict(lda=(1 << 22) + 16), "2^22 bytes apart"), (dict(m=(1 << 31) - 1, n=1 << 24, ldc=1 << 24), "too many tiles")]


@pytest.mark.parametrize("change,message", PRODUCT + [(dict(ldb=240), "pitch"), (dict(ld_bs=1), "pitch"), (dict(b_rows=64), "every row or every 128"), (dict(ldb=264), "16-byte"), (dict(workspace=4104), "workspace")])
def test_gemm_refuses_before_a_launch(change, message):
    _refused_product("cmx_fp8_block_gemm", {**GEMM, **change}, message)


@pytest.mark.parametrize("change,message", PRODUCT + [(dict(sizes=None), "null pointer"), (dict(groups=(1 << 20) + 1), "groups"), (dict(groups=0, zero_rest=1), "groups"),
                                                      (dict(k=(1 << 22) + 16, lda=(1 << 22) + 16, ld_as=1 << 16), "2^22 bytes apart")])
def test_gmm_refuses_before_a_launch(change, message):
    _refused_product("cmx_fp8_block_gmm", {**GMM, **change}, message)


def _refused_product(name, call, message):
    if message == "too many tiles" and not torch.cuda.is_available():
        assert getattr(_lib.load(), name)(*call.values()) < 0                    # (the number of CUs is asked for first)
        return
    _refused(name, call, message)


@pytest.mark.parametrize("name,call", [("cmx_fp8_block_quant", {**QUANT, **c}) for c in (dict(rows=0), dict(cols=0), dict(batch=0, x=None))] +
                         [("cmx_fp8_block_gemm", {**GEMM, **c}) for c in (dict(m=0), dict(n=0), dict(m=0, a=None))] +
                         [("cmx_fp8_block_gmm", {**GMM, **c}) for c in (dict(m=0), dict(n=0), dict(groups=0))])
def test_nothing_to_do_is_no_error(name, call):
    assert getattr(_lib.load(), name)(*call.values()) == 0
