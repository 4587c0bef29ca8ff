"""CPU: the paged key / value cache's argument checks, the bounds of its index arithmetic (csrc/paged_index.h compiled for the host), and the
oracle of its tests against a second formulation."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from oracle import paged_cpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _plan_args(R=3, W=4, N=20):
    return dict(lens=_i32(R), new=_i32(R), block_table=_i32(R, W), free_pages=_i32(N), num_free=_i32(1), page_size=16, width=2)


@pytest.mark.parametrize("change, match", [
    (dict(lens=torch.zeros(3, dtype=torch.int64)), "lens must be"), (dict(lens=_i32(4)), "lens must be"), (dict(new=_i32(3, 1)), "new must be"),
    (dict(block_table=_i32(3)), "block_table"), (dict(block_table=_i32(4, 3).t()), "block_table"), (dict(block_table=torch.zeros(3, 4)), "block_table"),
    (dict(block_table=_i32(1, 4).expand(3, 4)), "block_table"), (dict(block_table=_i32(3, 0)), "block_table"),
    (dict(free_pages=_i32(0)), "free_pages"), (dict(free_pages=_i32(40)[::2]), "free_pages"), (dict(num_free=_i32(2)), "num_free"),
    (dict(page_size=12), "power of two"), (dict(page_size=4), "power of two"), (dict(page_size=8192), "power of two"), (dict(width=0), "width"),
    (dict(lens_out=_i32(2)), "lens_out"), (dict(num_free_out=torch.zeros(1)), "num_free_out"), ({}, "only on an AMD GPU"),
])
def test_plan_refuses(change, match):
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import SpnError
    with pytest.raises(SpnError, match=match):
        ops.paged_plan(**{**_plan_args(), **change})


@pytest.mark.parametrize("change, match", [
    (dict(done=torch.zeros(3)), "done"), (dict(done=torch.zeros(2, dtype=torch.bool)), "done"), (dict(lens=_i32(5)), "lens"),
    (dict(page_size=24), "power of two"), ({}, "only on an AMD GPU"),
])
def test_release_refuses(change, match):
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import SpnError
    a = {k: v for k, v in _plan_args().items() if k not in ("new", "width")}
    with pytest.raises(SpnError, match=match):
        ops.paged_release(**{"done": torch.zeros(3, dtype=torch.bool), **a, **change})


def _pool(dtype=torch.bfloat16, kvh=2, page=16, d=64, n=5):
    return torch.zeros(n, kvh, page, d, dtype=dtype)


@pytest.mark.parametrize("change, match", [
    (dict(k=torch.zeros(4, 3, 64)), "k must be"), (dict(v=torch.zeros(3, 2, 64)), "v must be"), (dict(k=torch.zeros(4, 64, 2).transpose(1, 2)), "k must be"),
    (dict(k=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "one dtype"), (dict(slots=_i32(4)), "slots"), (dict(k_pages=_pool(d=32)), "k_pages"),
    (dict(v_pages=_pool(torch.float32)), "v_pages"), (dict(k_pages=_pool(page=12), v_pages=_pool(page=12)), "power of two"),
    (dict(k_pages=_pool(torch.float16), v_pages=_pool(torch.float16)), "unsupported dtype"), ({}, "only on an AMD GPU"),
])
def test_append_refuses(change, match):
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import SpnError
    a = dict(k=torch.zeros(4, 2, 64), v=torch.zeros(4, 2, 64), k_pages=_pool(), v_pages=_pool(), slots=torch.zeros(4, dtype=torch.int64))
    with pytest.raises(SpnError, match=match):
        ops.paged_append(**{**a, **change})


def test_append_refuses_one_memory_for_keys_and_values():
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import SpnError
    p = _pool()
    with pytest.raises(SpnError, match="same memory"):
        ops.paged_append(torch.zeros(4, 2, 64), torch.zeros(4, 2, 64), p, p, torch.zeros(4, dtype=torch.int64))


@pytest.mark.parametrize("change, match", [
    (dict(q=torch.zeros(3, 4, 64)), "q must be"), (dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), "q must be"), (dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), "q must be"),
    (dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), "3 heads on 2"), (dict(lens=_i32(2)), "lens"), (dict(slopes=torch.zeros(2)), "slopes"),
    (dict(slopes=torch.zeros(4, dtype=torch.bfloat16)), "slopes"), (dict(out=torch.zeros(3, 4, 64)), "out must be"),
    (dict(out=torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, 4, 64)), "out must be"),
    (dict(out=torch.zeros(3, 1, 64, dtype=torch.bfloat16).expand(3, 4, 64)), "out must be"),
    (dict(v_pages=_pool(n=6)), "v_pages"), (dict(k_pages=_pool().transpose(0, 1)), "k_pages"), ({}, "only on an AMD GPU"),
])
def test_attn_refuses(change, match):
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import SpnError
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k_pages=_pool(), v_pages=_pool(), block_table=_i32(3, 4), lens=_i32(3))
    with pytest.raises(SpnError, match=match):
        ops.paged_attn(**{**a, **change})


HOST_CHECK = r"""
#include "paged_index.h"
#include <cstdio>
#include <cstdlib>
#include <climits>
using namespace spn_paged;
#define NEED(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
static int odd() { static const int v[] = {0, 1, -1, 2, 7, 8, 9, 63, 64, 65, 100, 4095, 4096, 100000, INT_MAX, INT_MAX - 1, INT_MIN, INT_MIN + 1};
                   return std::rand() % 3 ? v[std::rand() % 18] : std::rand() % 5000 - 100; }
int main() {
    for (int it = 0; it < 2000000; ++it) {
        const int shift = 3 + std::rand() % 10, W = 1 + std::rand() % 300, pages = 1 + std::rand() % 1000, kvh = 1 + std::rand() % 8, width = 1 + std::rand() % 100;
        const int len = odd(), fresh = odd(), id = odd(), page = 1 << shift;
        const int n = rows_of(len, W, shift);
        NEED(n >= 0 && (n == 0 || n <= len) && (long)n <= (long)W << shift);
        NEED(n == 0 || ((n - 1) >> shift) < W);                                    // every row's table entry exists
        const int need = pages_needed(len, fresh, width, W, shift);
        if (need >= 0) {
            NEED(len >= 0 && fresh >= 0 && fresh <= width);
            NEED(pages_of(len, shift) + need <= W && ((long)len + fresh <= (long)W << shift));
            for (int i = 0; i < fresh; ++i) {                                       // each new row: an entry of the table row, held or taken
                const long pos = (long)len + i; const int j = (int)(pos >> shift), held = (int)pages_of(len, shift);
                NEED(j < W && (j < held || j - held < need));
                const long slot = slot_of(id, pos, pages, shift);
                NEED(slot == -1 ? !(id >= 0 && id < pages) : slot_ok(slot, pages, shift));
            }
        }
        const long slot = std::rand() % 2 ? (long)odd() : ((long)odd() << 20) + odd();
        if (slot_ok(slot, pages, shift)) {
            const long e = row_offset(slot >> shift, kvh - 1, slot & (page - 1), kvh, shift);
            NEED(e >= 0 && e + HEAD <= (long)pages * kvh * page * HEAD);
        }
        if (page_ok(id, pages)) {
            const long e = row_offset(id, std::rand() % kvh, page - 1, kvh, shift);
            NEED(e >= 0 && e + HEAD <= (long)pages * kvh * page * HEAD);
        }
    }
    // a pool past 2^32 elements
    NEED(row_offset(1 << 20, 7, 15, 8, 4) == (((1L << 20) * 8 + 7) * 16 + 15) * 64);
    std::puts("ok");
    return 0;
}
"""


def test_no_length_count_or_page_id_leads_outside_the_buffers(tmp_path):
    """The functions through which every device-side value becomes an address, over lengths, counts and ids of any value."""
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(HOST_CHECK)
    subprocess.run([shutil.which("g++") or "c++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "scoreperformer_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


def test_plan_and_release_oracle_are_inverse():
    rng = np.random.default_rng(0)
    for page in (8, 16):
        R, W, N = 9, 7, 80
        lens, table, stack = np.zeros(R, dtype=np.int32), np.full((R, W), -1, dtype=np.int32), [int(x) for x in rng.permutation(N)]
        new = rng.integers(0, W * page + 1, R)
        slots, lens, free = paged_cpu.plan(lens, new, table, stack, N, page, W * page)
        assert (lens == new).all() and len({int(s) for s in slots.flatten() if s >= 0}) == new.sum()
        before, tb, done = (lens.copy(), table.copy(), rng.random(R) < 0.5)
        after = paged_cpu.release(done, lens, table, stack, free, page)
        assert after - free == sum(paged_cpu.pages_of(int(n), page) for n in before[done])
        _, lens, again = paged_cpu.plan(lens, np.where(done, new, 0), table, stack, after, page, W * page)
        assert again == free and (table == tb).all() and (lens == before).all()


def test_attention_oracle_is_softmax_attention_of_the_gathered_rows():
    g = torch.Generator().manual_seed(0)
    R, h, kvh, page = 3, 4, 2, 8
    kp, vp = (torch.randn(10, kvh, page, 64, generator=g) for _ in range(2))
    q = torch.randn(R, h, 64, generator=g)
    table = torch.randperm(9, generator=g).int().view(R, 3)
    lens = torch.tensor([0, 5, 24])
    slopes = torch.tensor([0.5, 0.25, 0.0, 1.0])
    got = paged_cpu.attn(q, kp, vp, table, lens, slopes=slopes)
    assert (got[0] == 0).all()
    for r in (1, 2):
        n = int(lens[r])
        k, v = (p[table[r].long()].transpose(0, 1).flatten(1, 2)[:, :n].double().repeat_interleave(2, 0) for p in (kp, vp))
        s = torch.einsum("hjd,hd->hj", k, q[r].double()) / 8 + slopes.double()[:, None] * torch.arange(-n + 1, 1).double()
        want = torch.einsum("hj,hjd->hd", torch.exp(s) / torch.exp(s).sum(1, keepdim=True), v)
        assert (got[r] - want).abs().max() < 1e-12


def _stack(**kw):
    from scoreperformer_amd.modules.transformer import Decoder
    return Decoder(dim=64, depth=2, heads=1, **kw).eval()


def test_paged_cache_refuses_what_it_does_not_serve():
    from scoreperformer_amd.modules.transformer import AttentionConfig, Encoder, PagedKVCache
    ok = dict(num_pages=4, max_requests=2, max_len=20)
    c = PagedKVCache(_stack(), **ok)
    assert c.k_pages.shape == (2, 4, 1, 16, 64) and c.block_table.shape == (2, 2) and int(c.num_free) == 4 and c.k_pages.dtype == torch.bfloat16
    with pytest.raises(NotImplementedError, match="causal"):
        PagedKVCache(Encoder(dim=64, depth=2, heads=1), **ok)
    with pytest.raises(NotImplementedError, match="cross"):
        PagedKVCache(_stack(cross_attend=True), **ok)
    with pytest.raises(NotImplementedError, match="memory"):
        PagedKVCache(_stack(attention=AttentionConfig(num_mem_kv=2)), **ok)
    for new in (torch.ones(1, dtype=torch.int32), torch.ones(2, 1, dtype=torch.int32)):     # (would broadcast)
        with pytest.raises(ValueError, match="new rows"):
            c.plan(new, width=4)
    for bad in (dict(num_pages=0), dict(max_requests=0), dict(max_len=0), dict(page_size=12), dict(page_size=4)):
        with pytest.raises(ValueError):
            PagedKVCache(_stack(), **{**ok, **bad})


def test_paged_steps_refuse_masks_gradients_and_other_stacks():
    from scoreperformer_amd.modules.transformer import AttentionConfig, PagedKVCache, PagedStep
    stack = _stack(attention=AttentionConfig(one_kv_head=True))
    cache = PagedKVCache(stack, num_pages=4, max_requests=2, max_len=20)
    step = PagedStep(cache, torch.zeros(2, 1, dtype=torch.int64), torch.ones(2, 1, dtype=torch.bool), torch.ones(2, dtype=torch.int32))
    x = torch.zeros(2, 1, 64)
    with pytest.raises(ValueError, match="own mask"):
        stack(x, mask=torch.ones(2, 1, dtype=torch.bool), paged=step)
    with pytest.raises(ValueError, match="layers"):
        _stack().__class__(dim=64, depth=3, heads=1)(x, paged=step)
    attn = stack.layers[0][1]
    with pytest.raises(ValueError, match="no context"):
        attn(x, mask=step.mask, paged=(step, 0))
    with pytest.raises(RuntimeError, match="inference"):
        attn(x, paged=(step, 0))
    with torch.no_grad():
        with pytest.raises(ValueError, match="do not fit"):
            attn(torch.zeros(3, 1, 64), paged=(step, 0))
        attn.train()
        with pytest.raises(RuntimeError, match="inference"):
            attn(x, paged=(step, 0))
