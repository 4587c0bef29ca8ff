"""CPU: more calls of the paged cache that are refused by the wrappers' own error, before anything runs."""
import pytest
import torch

BF16 = torch.bfloat16


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("out", [torch.zeros(12, 64, dtype=BF16), torch.zeros(1, 3, 4, 64, dtype=BF16), torch.zeros((), dtype=BF16), torch.zeros(0, dtype=BF16)])
def test_attention_refuses_an_output_of_another_rank(out):
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import SpnError
    pool = torch.zeros(5, 2, 16, 64, dtype=BF16)
    with pytest.raises(SpnError, match="out must be like q"):
        ops.paged_attn(torch.zeros(3, 4, 64, dtype=BF16), pool, pool.clone(), _i32(3, 4), _i32(3), out=out)
