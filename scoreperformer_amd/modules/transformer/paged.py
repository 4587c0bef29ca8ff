"""Paged key / value cache of a decoder stack: many requests of different, growing lengths in one batch.

The reference's cached decode (`modules/transformer/attention.py:155-156`, `transformer.py:160-195`) concatenates every layer's keys, values and
hidden states with the new row each step, for a batch whose sequences all have the same length.  Here a request's rows live in pages of one
pool per layer, found through a block table; a step appends one row per request in place and attends over the pages
(`ops.paged_plan / paged_append / paged_attn / paged_release`).  Nothing is read back to the host, so a step can be captured in a hipGraph.

    cache = PagedKVCache(decoder, num_pages=4096, max_requests=64, max_len=2048)
    step = cache.plan(prompt_lengths, width=n)             # prompts of requests that hold nothing yet: x [max_requests, n, dim], right-padded
    hidden = decoder(x, paged=step)
    step = cache.plan(active)                              # one more row for the requests with active[r] = 1 (int32)
    hidden = decoder(x_new, paged=step)                    # x_new [max_requests, 1, dim]
    cache.release(done)                                    # done [max_requests] bool: pages go back, the rows of the batch are free for others
"""
from dataclasses import dataclass
from typing import Optional

import torch
from torch import Tensor

from ... import ops


@dataclass
class PagedStep:
    """The rows of one forward pass: where they go (slots [R, width], -1: no row), which of them there are (mask) and, for single rows, how many each
    of the requests with a row now holds (lens [R], the new one included; 0: no row this time)."""
    cache: "PagedKVCache"
    slots: Tensor
    mask: Tensor
    lens: Optional[Tensor]

    @property
    def width(self) -> int:
        return self.slots.shape[1]


class PagedKVCache:
    """`stack`: the decoder (`Transformer`, causal, self-attention only) whose layers it serves.  One pool of `num_pages` pages of `page_size` rows per
    layer, the same page ids for all layers; `max_len`: rows a request can hold, rounded up to whole pages; bf16, like the operands of the attention kernels."""

    def __init__(self, stack, num_pages: int, max_requests: int, max_len: int, page_size: int = 16, device=None):
        blocks = [layer[1] for kind, layer in zip(stack.layer_types, stack.layers) if kind == "a"]
        if stack.cross_attend or not blocks or any(not b.causal or b.num_mem_kv for b in blocks):
            raise NotImplementedError("PagedKVCache serves causal self-attention stacks without cross-attention or learned memory keys")
        if num_pages < 1 or max_requests < 1 or max_len < 1:
            raise ValueError("num_pages, max_requests and max_len must be positive")
        if page_size < 8 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"the page size must be a power of two in [8, 4096], got {page_size}")
        device = torch.device(device) if device is not None else blocks[0].to_q.weight.device
        self.page_size, self.kv_heads, self.num_layers = page_size, blocks[0].kv_heads, len(blocks)
        ints = dict(device=device, dtype=torch.int32)
        self.k_pages, self.v_pages = (torch.zeros(len(blocks), num_pages, self.kv_heads, page_size, ops.PAGED_HEAD, device=device, dtype=torch.bfloat16)
                                      for _ in range(2))
        self.block_table = torch.full((max_requests, -(-max_len // page_size)), -1, **ints)
        self.lens = torch.zeros(max_requests, **ints)
        self.free_pages, self.num_free = torch.arange(num_pages, **ints), torch.full((1,), num_pages, **ints)

    @property
    def max_requests(self) -> int:
        return self.lens.shape[0]

    @torch.no_grad()
    def plan(self, new: Tensor, width: int = 1) -> PagedStep:
        """Room for new [R] (int32, on the device) more rows per request, at most `width` each.  width > 1 is the prompt form: its rows attend to each
        other only, so a request that already holds rows takes none (its count is refused).  A request that cannot be served whole -- no pages left,
        more than `max_len` rows -- takes none either: its slots are -1, its length stays, and the attention adds nothing to its rows (step.mask tells)."""
        if new.shape != self.lens.shape:
            raise ValueError(f"new rows of {list(new.shape)} for {self.max_requests} requests")
        if width > 1:
            new = torch.where((self.lens == 0) | (new == 0), new, -1)
        slots, _, _ = ops.paged_plan(self.lens, new, self.block_table, self.free_pages, self.num_free, self.page_size, width, lens_out=self.lens,
                                     num_free_out=self.num_free)
        mask = slots >= 0
        return PagedStep(self, slots, mask, torch.where(mask[:, 0], self.lens, 0) if width == 1 else None)

    @torch.no_grad()
    def release(self, done: Tensor) -> None:
        """The requests with done [R] (bool, on the device) give their pages back and hold nothing."""
        ops.paged_release(done, self.lens, self.block_table, self.free_pages, self.num_free, self.page_size)

    def append(self, layer: int, k: Tensor, v: Tensor, step: PagedStep) -> None:
        """Rows k, v [R * width, kv_heads, 64] of `layer` into the step's slots."""
        ops.paged_append(k, v, self.k_pages[layer], self.v_pages[layer], step.slots)

    def attend(self, layer: int, q: Tensor, step: PagedStep, scale: float, slopes: Optional[Tensor] = None) -> Tensor:
        """q [R, heads, 64] of a single-row step over the rows that `layer` holds, the appended ones among them."""
        return ops.paged_attn(q, self.k_pages[layer], self.v_pages[layer], self.block_table, step.lens, scale=scale, slopes=slopes)
