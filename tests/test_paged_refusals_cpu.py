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


@pytest.mark.parametrize("k_at, v_at", [(0, 1), (1, 0), (0, 4), (2, 2)])
def test_append_refuses_pools_that_overlap(k_at, v_at):
    """Slices of one pool that share pages: a row's key and another's value would go to one place."""
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import SpnError
    pool, rows = torch.zeros(10, 2, 16, 64), torch.zeros(4, 2, 64)
    slots = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(SpnError, match="same memory"):
        ops.paged_append(rows, rows, pool[k_at:k_at + 5], pool[v_at:v_at + 5], slots)
    with pytest.raises(SpnError, match="only on an AMD GPU"):       # side by side: accepted
        ops.paged_append(rows, rows, pool[:5], pool[5:], slots)
