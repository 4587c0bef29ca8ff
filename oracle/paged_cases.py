"""Inputs of the accuracy tests of the paged attention (tests/test_paged_accuracy_{cpu,gpu}.py): the same for arithmetic in other precisions on the CPU
and for the kernels."""
import numpy as np
import torch

BF16, F32 = torch.bfloat16, torch.float32

# heads, key heads, page, lengths, slope of the first head (0: no bias)
CASES = {
    "tile edges": (8, 1, 16, [2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129], 0.0),
    "ragged": (6, 3, 8, [1000, 40, 1537, 30], 0.02),
    "passes": (20, 1, 128, [500, 77, 260], 0.01),
    "long": (8, 2, 16, [5003], 0.0),
    "cut": (4, 1, 32, [131, 40000, 70], 0.0),
    "many": (8, 8, 16, [(i * 37) % 301 + 20 for i in range(40)], 0.05),
}


def slopes_of(case):
    h, first = CASES[case][0], CASES[case][4]
    return torch.tensor([first * 2.0 ** (-8.0 * i / h) for i in range(h)]) if first else None


def make(case, dtype, cancel=False):
    """(q, k_pages, v_pages, table, lens) on the CPU.  cancel: values of +-1, as many of either sign in every dimension, under scores that differ
    little: what the weights lose in rounding is what the output shows."""
    h, kvh, page, lens, _ = CASES[case]
    g, rng = torch.Generator().manual_seed(len(case)), np.random.default_rng(len(case))
    held = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(held) + 2)
    table = np.full((len(lens), max(held)), -1, dtype=np.int64)
    kp, vp = (torch.full((len(ids), kvh, page, 64), float("nan")) for _ in range(2))
    at = 0
    for r, n in enumerate(lens):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
        rows = torch.from_numpy(table[r, :held[r]]).repeat_interleave(page)[:n], torch.arange(n) % page
        k, v = torch.randn(n, kvh, 64, generator=g), torch.randn(n, kvh, 64, generator=g)
        if cancel:
            sign = torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
            v = torch.stack([sign[torch.randperm(n, generator=g)] for _ in range(kvh * 64)], 1).view(n, kvh, 64)
        kp[rows[0], :, rows[1]], vp[rows[0], :, rows[1]] = k, v
    q = torch.randn(len(lens), h, 64, generator=g) * (0.5 if cancel else 1.0)
    return q.to(dtype), kp.to(dtype), vp.to(dtype), torch.from_numpy(table).int(), torch.tensor(lens, dtype=torch.int32)
