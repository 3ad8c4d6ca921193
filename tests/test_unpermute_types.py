"""The weighted way back reads bf16 rows, fp32 weights and an int32 table of routes: anything else is refused, on the host, before a device is looked at."""
import pytest
import torch

from catccos_amd import ops

ROWS, TO, PROBS = torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2)


@pytest.mark.parametrize("y,to,probs", [
    (ROWS.half(), TO, PROBS), (ROWS.float(), TO, PROBS), (ROWS.view(torch.uint8), TO, PROBS), (ROWS.t().contiguous().t(), TO, PROBS), (ROWS[:, ::2], TO, PROBS),
    (ROWS, TO.long(), PROBS), (ROWS, TO.float(), PROBS), (ROWS, TO[:-1], PROBS), (ROWS, torch.cat([TO, TO]), PROBS), (ROWS, torch.cat([TO, TO])[::2], PROBS),
    (ROWS, TO, PROBS.half()), (ROWS, TO, PROBS.double()), (ROWS, TO, torch.zeros(2, 4).t()), (ROWS, TO, PROBS[:, :0])])
def test_other_types_and_layouts_are_refused(y, to, probs):
    with pytest.raises(AssertionError):
        ops.moe_token_unpermute(y, to, probs)


@pytest.mark.parametrize("y", [ROWS, ROWS.view(torch.int16), ROWS.view(torch.uint16), torch.zeros(8, 20, dtype=torch.bfloat16)[:, :16]])
def test_what_it_reads_gets_as_far_as_the_device(y):
    with pytest.raises(ValueError, match="expected a GPU tensor"):
        ops.moe_token_unpermute(y, TO, PROBS)
    with pytest.raises(ValueError, match="expected a GPU tensor"):
        ops.moe_token_unpermute(y, TO.view(4, 2), PROBS)
