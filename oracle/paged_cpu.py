"""CPU restatement of the paged key / value cache (scoreperformer_amd.ops.paged_*) -- TEST INFRASTRUCTURE, not product code.

Written request by request, with Python lists and 64-bit floats, from the definitions only: the reference has no paged cache (it
concatenates caches per step, modules/transformer/attention.py:155-156), so parity is to the formulas and, for the attention, to the
reference's own dense attention on the same rows (oracle/ref_cpu.py through tests/test_paged_module_gpu.py)."""
from typing import List, Optional

import numpy as np
import torch

HEAD = 64


def pages_of(n: int, page: int) -> int:
    return -(-n // page) if n > 0 else 0


def plan(lens, new, table: np.ndarray, stack: List[int], num_free: int, page: int, width: int):
    """table is changed in place; returns (slots, lens, num_free).  `stack`: the whole array of num_pages entries."""
    num_pages = len(stack)
    num_free = min(max(num_free, 0), num_pages)
    lens, slots, asked, taken = list(lens), np.full((len(lens), width), -1, dtype=np.int64), 0, 0
    for r in range(len(lens)):
        n = int(new[r])
        if lens[r] < 0 or not 0 <= n <= width or pages_of(lens[r] + n, page) > table.shape[1]:
            continue
        held, after = pages_of(lens[r], page), pages_of(lens[r] + n, page)
        asked += after - held
        if after > held and asked > num_free:
            continue
        for j in range(held, after):
            table[r, j] = stack[num_free - 1 - taken]
            taken += 1
        for i in range(n):
            pos = lens[r] + i
            pid = int(table[r, pos // page])
            slots[r, i] = pid * page + pos % page if 0 <= pid < num_pages else -1
        lens[r] += n
    return slots, np.asarray(lens, dtype=np.int32), num_free - taken


def release(done, lens, table: np.ndarray, stack: List[int], num_free: int, page: int):
    """lens, table, stack are changed in place; returns num_free."""
    num_pages = len(stack)
    num_free = min(max(num_free, 0), num_pages)
    back = []
    for r in range(len(lens)):
        if done[r]:
            held = min(pages_of(int(lens[r]), page), table.shape[1])
            back += [int(p) for p in table[r, :held] if 0 <= p < num_pages]
            table[r, :held] = -1
            lens[r] = 0
    for i, p in enumerate(reversed(back)):
        if num_free + i < num_pages:
            stack[num_free + i] = p
    return min(num_free + len(back), num_pages)


def append(rows: torch.Tensor, pages: torch.Tensor, slots: torch.Tensor) -> None:
    """In place on `pages` [num_pages, kvh, page, 64]; rows [T, kvh, 64]."""
    page = pages.shape[2]
    for t, s in enumerate(slots.flatten().tolist()):
        if 0 <= s < pages.shape[0] * page:
            pages[s // page, :, s % page] = rows[t].to(pages.dtype)


def attn(q, k_pages, v_pages, table, lens, scale: Optional[float] = None, slopes=None):
    """64-bit [R, h, 64] from CPU tensors."""
    R, h, d = q.shape
    num_pages, kvh, page, _ = k_pages.shape
    scale = HEAD ** -0.5 if scale is None else scale
    out = torch.zeros(R, h, d, dtype=torch.float64)
    for r in range(R):
        n = min(max(int(lens[r]), 0), table.shape[1] * page)
        ks, vs, js = [], [], []
        for j0 in range(0, n, page):
            pid = int(table[r, j0 // page])
            if 0 <= pid < num_pages:
                m = min(page, n - j0)
                ks.append(k_pages[pid, :, :m].double()); vs.append(v_pages[pid, :, :m].double()); js.append(torch.arange(j0, j0 + m))
        if not ks:
            continue
        k, v, j = torch.cat(ks, 1), torch.cat(vs, 1), torch.cat(js)
        for hi in range(h):
            s = scale * (k[hi * kvh // h] @ q[r, hi].double())
            if slopes is not None:
                s = s - float(slopes[hi]) * (n - 1 - j).double()
            p = torch.softmax(s, 0)
            out[r, hi] = p @ v[hi * kvh // h]
    return out


def attn_and_bound(q, k_pages, v_pages, table, lens, scale: Optional[float] = None, slopes=None):
    """`attn` and, element by element, how far 32-bit arithmetic may be from it (u = 2^-24, w the weights of a request's rows under one head).

    A score: its 64 products sum to A in absolute value; 64 roundings of partial sums that are independent and at most A give 8 u A (their worst case,
    64 u A, needs every partial sum at A and every rounding to one side); scale, slope and their products are rounded a few times each, the running
    reference (at most 6 from the largest score) whenever it moves.  The exponential is off by one unit in the last place and by its argument's
    rounding.  Together a relative error d_j of every weight, which moves the output by at most sum_j w_j d_j (|v_j| + |o|).  Sums over n rows:
    independent roundings again, 2 sqrt(n) u of the absolute terms, and 16 u for joining waves and parts, in numerator and denominator.
    bf16 pools: a weight that enters the product as two bf16 terms keeps 2^-16 of itself, and the output is rounded once (2^-8; fp32: u)."""
    u, bf = 2.0 ** -24, q.dtype == torch.bfloat16
    R, h, d = q.shape
    num_pages, kvh, page, _ = k_pages.shape
    scale = HEAD ** -0.5 if scale is None else scale
    out, tol = (torch.zeros(R, h, d, dtype=torch.float64) for _ in range(2))
    for r in range(R):
        n = min(max(int(lens[r]), 0), table.shape[1] * page)
        ids = table[r, :pages_of(n, page)].long()
        there = ((ids >= 0) & (ids < num_pages)).repeat_interleave(page)[:n]
        j = torch.arange(n)[there]
        if len(j) == 0:
            continue
        rows = ids[j // page] * page + j % page
        k, v = (p.transpose(1, 2).reshape(-1, kvh, d)[rows].double() for p in (k_pages, v_pages))       # [rows, kvh, d]
        dist = (n - 1 - j).double()
        for hi in range(h):
            kh, vh = k[:, hi * kvh // h], v[:, hi * kvh // h]
            slope = float(slopes[hi]) if slopes is not None else 0.0
            products = scale * kh * q[r, hi].double()
            s, bias = products.sum(1), slope * dist
            x = s - bias
            top = x.max()
            w = torch.softmax(x, 0)
            o = w @ vh
            rel = u * (8 * products.abs().sum(1) + 4 * s.abs() + 4 * bias.abs() + 60 * abs(slope) + 6 * (top.abs() + 6) + (x - top).abs() + 4)
            if bf:
                rel = rel + 2.0 ** -16
            out[r, hi] = o
            tol[r, hi] = (w * rel) @ (vh.abs() + o.abs()) + 2 * (16 + 2 * len(j) ** 0.5) * u * (w @ vh.abs()) + o.abs() * (2.0 ** -8 if bf else u)
    return out, tol
