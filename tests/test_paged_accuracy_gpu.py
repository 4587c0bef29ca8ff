"""GPU: the paged attention within what 32-bit arithmetic (bf16 pools: with weights of two bf16 terms, rounded once at the end) may be off, element by
element; tests/test_paged_accuracy_cpu.py shows on the same inputs that fewer bits fail this bound."""
import pytest
import torch

from oracle import paged_cpu
from oracle.paged_cases import BF16, CASES, F32, make, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("wide", [0, 20000])
def test_attention_is_as_near_as_its_arithmetic(dev, case, cancel, dtype, wide):
    """In tables of the batch's own width and in far wider ones (whole segments and cut ones)."""
    from scoreperformer_amd import ops
    q, kp, vp, table, lens = make(case, dtype, cancel)
    slopes = slopes_of(case)
    want, tol = paged_cpu.attn_and_bound(q, kp, vp, table, lens, slopes=slopes)
    table = torch.nn.functional.pad(table, (0, wide // kp.shape[2]), value=-1)
    got = ops.paged_attn(*(t.to(dev) for t in (q, kp, vp, table, lens)), slopes=None if slopes is None else slopes.to(dev)).cpu().double()
    ratio = (got - want).abs() / tol
    assert bool((ratio <= 1).all()), float(ratio.max())
