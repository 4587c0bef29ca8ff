"""CPU: the element-wise bound of the paged attention's accuracy tests (oracle/paged_cpu.py attn_and_bound) lets 32-bit arithmetic pass and fails
arithmetic in fewer bits, on the very inputs that the GPU tests use."""
import pytest
import torch

from oracle import paged_cpu
from oracle.paged_cases import BF16, CASES, F32, make, slopes_of


def _attention(q, kp, vp, table, lens, slopes, weights, operands=F32):
    """In 32 bits, with operands (queries, keys) and weights put through a rounding of the caller's."""
    R, h, d = q.shape
    kvh, page = kp.shape[1:3]
    out = torch.zeros(R, h, d)
    for r in range(R):
        n = int(lens[r])
        ids = table[r, :-(-n // page)].long()
        k, v = (p[ids].transpose(0, 1).flatten(1, 2)[:, :n].to(operands if i == 0 else p.dtype).float() for i, p in enumerate((kp, vp)))
        for hi in range(h):
            s = (k[hi * kvh // h] @ q[r, hi].to(operands).float()) * 0.125
            if slopes is not None:
                s = s - slopes[hi] * torch.arange(n - 1, -1, -1)
            p = weights(torch.exp(s - s.max()))
            out[r, hi] = (p @ v[hi * kvh // h]) / p.sum()
    return out


def _two_terms(p):
    hi = p.to(BF16).float()
    return hi + (p - hi).to(BF16).float()


def _worst(case, dtype, cancel, weights, operands=F32):
    data = make(case, dtype, cancel)
    want, tol = paged_cpu.attn_and_bound(*data, slopes=slopes_of(case))
    got = _attention(*data, slopes_of(case), weights, operands).to(dtype).double()
    return float(((got - want).abs() / tol).max())


def same(p):
    return p


def once(p):
    return p.to(BF16).float()


@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("case", list(CASES))
def test_the_bound_holds_for_32_bits_and_fails_for_fewer(case, cancel):
    assert _worst(case, F32, cancel, same) <= 0.5
    assert _worst(case, F32, cancel, once) > 1.5                       # weights in bf16
    assert _worst(case, F32, cancel, same, operands=BF16) > 1.5        # queries and keys in bf16
    assert _worst(case, BF16, cancel, _two_terms) <= 1.0               # (ordinary values: the output's rounding alone comes up to 1)
    if cancel:
        assert _worst(case, BF16, cancel, once) > 1.5                  # bf16 pools, the weights' second term left out


@pytest.mark.parametrize("case", ["tile edges", "ragged"])
def test_the_bound_belongs_to_the_oracle(case):
    data = make(case, F32)
    want, _ = paged_cpu.attn_and_bound(*data, slopes=slopes_of(case))
    assert float((want - paged_cpu.attn(*data, slopes=slopes_of(case))).abs().max()) < 1e-12
