"""Cases of the paged key / value cache: block tables and slot maps built on the GPU, new rows written into the pages, and the attention
of one new note per request over them.  Layouts: pages [num_pages, kv_heads, page, 64]; block_table [requests, width] int32 (-1: no page);
lens [requests] int32; the free pages are a stack of page ids (free_pages [num_pages], num_free [1]).

`run` computes the operators with elementary torch operations, or (own = True) with scoreperformer_amd.ops."""
import math

import numpy as np
import torch

own = False

HEAD = 64    # the attention kernels' head width
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # a decode step of a serving batch: every request gets one more note
        dict(name="plan, one note for each of 64", op="plan", requests=64, longest=4096, shortest=1, page=16, width=1),
        # the prompts of a batch arrive at once (render windows of up to 2048 notes)
        dict(name="plan, prompts of 64", op="plan", requests=64, longest=0, shortest=0, page=16, width=2048),
        # half of a large batch has ended: its pages go back and new prompts of the same lengths take them
        dict(name="turnover, half of 510", op="turnover", requests=510, longest=1024, shortest=1, page=16, width=1024),
        # a decode step's rows: one key / value row per request, out of the fused projection buffer
        dict(name="append, one note for each of 64", op="append", requests=64, width=1, heads=8, kv_heads=1, page=16, rows="bf16", pages="bf16"),
        # a batch of prompts, multi-head keys, fp32 rows rounded on the way in
        dict(name="append, prompts of 64 x 1024", op="append", requests=64, width=1024, heads=8, kv_heads=8, page=16, rows="fp32", pages="bf16"),
        # one performance being rendered, 4096 notes, multi-query heads: latency
        dict(name="attn, 1 x 4096, multi-query", op="attn", requests=1, longest=4096, shortest=4096, heads=8, kv_heads=1, page=16, dtype="bf16", alibi=True),
        # an ordinary ragged serving batch of the default decoder; one request is still empty
        dict(name="attn, 64 x 0..2048, multi-query", op="attn", requests=64, longest=2048, shortest=0, heads=8, kv_heads=1, page=16, dtype="bf16", alibi=True),
        # the decode engine's precision
        dict(name="attn, 32 x 1..4096, fp32", op="attn", requests=32, longest=4096, shortest=1, heads=8, kv_heads=1, page=16, dtype="fp32", alibi=True),
        # odd sizes, three key heads, no positional bias
        dict(name="attn, 13 x 1..1001, 6 on 3 heads", op="attn", requests=13, longest=1001, shortest=1, heads=6, kv_heads=3, page=8, dtype="fp32", alibi=False),
        # grouped heads, large pages
        dict(name="attn, 128 x 1..8192, 8 on 2 heads", op="attn", requests=128, longest=8192, shortest=1, heads=8, kv_heads=2, page=64, dtype="bf16", alibi=True),
        # a few very long caches
        dict(name="attn, 4 x 100..131072", op="attn", requests=4, longest=131072, shortest=100, heads=8, kv_heads=1, page=32, dtype="bf16", alibi=True),
        # a full machine: multi-head keys, 256 requests
        dict(name="attn, 256 x 1..4096, multi-head", op="attn", requests=256, longest=4096, shortest=1, heads=8, kv_heads=8, page=16, dtype="bf16", alibi=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "turnover", "append", "attn", "attn", "attn", "attn"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "plan":
        if rng.random() < 0.5:     # a decode step
            return dict(op=op, requests=_log(rng, 1, 2048), longest=_log(rng, 64, 8192), shortest=rng.choice([0, 1]), page=page, width=1)
        return dict(op=op, requests=_log(rng, 1, 256), longest=rng.choice([0, _log(rng, 1, 2048)]), shortest=0, page=page, width=_log(rng, 2, 2048))
    if op == "turnover":
        longest = _log(rng, 16, 2048)
        return dict(op=op, requests=_log(rng, 2, 1024), longest=longest, shortest=rng.choice([0, 1]), page=page, width=longest)
    kv_heads, group = rng.choice([(1, 8), (1, 8), (1, 5), (1, 16), (1, 24), (2, 4), (3, 2), (4, 3), (8, 1), (8, 1), (6, 1)])
    if op == "append":
        return dict(op=op, requests=_log(rng, 1, 512), width=rng.choice([1, _log(rng, 2, 128)]), heads=group * kv_heads, kv_heads=kv_heads, page=page,
                    rows=rng.choice(["bf16", "fp32"]), pages=rng.choice(["bf16", "fp32"]))
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    requests = _log(rng, 1, 256)
    most = 256 * 4096 * 8 * 2 // (requests * kv_heads * SIZE[dtype])      # the padded extent of the largest listed case, in bytes
    longest = _log(rng, 1, min(131072, most))
    return dict(op=op, requests=requests, longest=longest, shortest=rng.choice([0, 1, longest // 2, longest]), heads=group * kv_heads, kv_heads=kv_heads,
                page=page, dtype=dtype, alibi=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------------------------------ inputs

def _spread(lo, hi, n):
    """n lengths evenly over lo .. hi, both ends among them: the same total for every seed."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case):
    """(cached notes, new notes) of the case's requests, in the order before the seed's shuffle."""
    n = case["requests"]
    if case["op"] == "attn":
        return _spread(case["shortest"], case["longest"], n), [0] * n
    if case["op"] == "append":
        return [0] * n, _spread(1, case["width"], n)
    cached = _spread(case["shortest"], case["longest"], n)
    if case["op"] == "plan":
        return cached, _spread(1, case["width"], n)[::-1]
    return cached, [c if i % 2 else 0 for i, c in enumerate(cached)]     # turnover: the odd ones end and come again


def _pages_of(length, page):
    return -(-length // page)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 32)).permutation(case["requests"])
    cached, new = (np.asarray(x, dtype=np.int64)[order] for x in _lengths(case))
    page = case["page"]
    room = cached + (new if case["op"] != "turnover" else 0)
    width = max(1, int(max(_pages_of(int(x), page) for x in room)))
    held = -(-cached // page)
    num_pages = int(sum(_pages_of(int(x), page) for x in room)) + 8
    ids = np.random.RandomState((seed + 1) % (1 << 32)).permutation(num_pages).astype(np.int32)
    table = np.full((case["requests"], width), -1, dtype=np.int32)
    table[np.arange(width)[None, :] < held[:, None]] = ids[:held.sum()]
    stack = np.zeros(num_pages, dtype=np.int32)
    stack[:num_pages - held.sum()] = ids[held.sum():]

    def up(a, dtype):
        return torch.from_numpy(np.ascontiguousarray(a)).to(device=dev, dtype=dtype)

    s = dict(case=case, page=page, width=case.get("width", 1), table=up(table, torch.int32), lens=up(cached, torch.int32), new=up(new, torch.int32),
             free=up(stack, torch.int32), num_free=up([num_pages - held.sum()], torch.int32))
    if case["op"] == "turnover":
        s["done"] = up((cached == new) & (new > 0), torch.bool)
        return s
    if case["op"] == "plan":
        return s
    kvh, h = case["kv_heads"], case["heads"]
    dtype = DTYPES[case["pages" if case["op"] == "append" else "dtype"]]
    s["k_pages"], s["v_pages"] = (torch.randn(num_pages, kvh, page, HEAD, device=dev, generator=g).to(dtype) for _ in range(2))
    if case["op"] == "append":
        n = case["requests"] * case["width"]
        rows = torch.randn(n, (h + 2 * kvh) * HEAD, device=dev, generator=g).to(DTYPES[case["rows"]])     # q | k | v, as the fused projection leaves them
        s["k"], s["v"] = (rows[:, a * HEAD:(a + kvh) * HEAD].unflatten(1, (kvh, HEAD)) for a in (h, h + kvh))
        at = np.arange(case["width"])[None, :]
        first = np.cumsum(-(-new // page)) - (-(-new // page))
        pages = ids[np.minimum(first[:, None] + at // page, num_pages - 1)].astype(np.int64)
        s["slots"] = up(np.where(at < new[:, None], pages * page + at % page, -1), torch.int64)
        return s
    # rows of the last page behind a request's length hold whatever was there: here, no numbers
    some = np.nonzero((cached % page) > 0)[0]
    rest = [(table[r, held[r] - 1], o) for r in some for o in range(cached[r] % page, page)]
    if rest:
        pg, off = (up([x[i] for x in rest], torch.int64) for i in (0, 1))
        for pool in (s["k_pages"], s["v_pages"]):
            pool[pg, :, off] = float("nan")
    s["q"] = torch.randn(case["requests"], h, HEAD, device=dev, generator=g).to(dtype)
    # geometric slopes, as ALiBi has them
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device=dev) if case["alibi"] else None
    return s


# ------------------------------------------------------------------------------------------------------------- the plain forms

def _release(s):
    """Pages of the ended requests go back on the stack, so that the first page of the first request lies on top."""
    table, lens, free, num_free = s["table"], s["lens"], s["free"], s["num_free"]
    at = torch.arange(table.shape[1], device=table.device)
    held = (lens.long() + s["page"] - 1) // s["page"]
    back = s["done"][:, None] & (at < held[:, None]) & (table >= 0) & (table < free.numel())
    rank = torch.cumsum(back.flatten().long(), 0)
    top = num_free.long() + rank[-1:]
    where = torch.where(back.flatten(), top - rank, free.numel())
    grown = torch.cat([free, free.new_zeros(1)])
    grown[where] = table.flatten()
    free.copy_(grown[:-1])
    num_free.copy_(top)
    table.copy_(torch.where(s["done"][:, None] & (at < held[:, None]), -1, table))
    lens.copy_(torch.where(s["done"], 0, lens))


def _plan(s):
    table, page, free, width = s["table"], s["page"], s["free"], s["width"]
    lens, new = s["lens"].long(), s["new"].long()
    at = torch.arange(table.shape[1], device=table.device)
    held, after = (lens + page - 1) // page, (lens + new + page - 1) // page
    fits = (new >= 0) & (new <= width) & (lens >= 0) & (after <= table.shape[1])
    need = torch.where(fits, after - held, 0)
    end = torch.cumsum(need, 0)
    given = fits & ((need == 0) | (end <= s["num_free"]))
    first = s["num_free"] - 1 - (end - need)
    fresh = given[:, None] & (at >= held[:, None]) & (at < after[:, None])
    taken = free[(first[:, None] - (at - held[:, None])).clamp(0, free.numel() - 1)]
    table.copy_(torch.where(fresh, taken, table))
    i = torch.arange(width, device=table.device)
    pos = lens[:, None] + i
    ids = torch.gather(table, 1, (pos // page).clamp(0, table.shape[1] - 1)).long()
    live = given[:, None] & (i < new[:, None]) & (ids >= 0) & (ids < free.numel())
    slots = torch.where(live, ids * page + pos % page, -1)
    return slots, (lens + torch.where(given, new, 0)).int(), (s["num_free"] - torch.where(given, need, 0).sum()).int()


def _append(s):
    for rows, pool in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        slots = s["slots"].flatten()
        live = slots >= 0
        to = torch.where(live, slots, slots.numel() and slots.max())           # a row without a slot repeats the last one's ...
        src = torch.where(live, torch.arange(slots.numel(), device=slots.device), slots.argmax())
        pool[to // s["page"], :, to % s["page"]] = rows[src].to(pool.dtype)      # ... with its values
    return s["k_pages"], s["v_pages"]


def _attn(s):
    q, table, page = s["q"].float(), s["table"].long(), s["page"]
    r, h, d = q.shape
    kvh = s["k_pages"].shape[1]
    key = torch.arange(table.shape[1] * page, device=q.device)
    ids = table[:, key // page]
    live = (key < s["lens"][:, None]) & (ids >= 0)
    k, v = (pool[ids.clamp(min=0), :, key % page].permute(0, 2, 1, 3).float() for pool in (s["k_pages"], s["v_pages"]))     # [r, kvh, keys, d]
    scores = torch.matmul(q.view(r, kvh, h // kvh, d), k.transpose(2, 3)).view(r, h, -1) * d ** -0.5
    if s["slopes"] is not None:
        scores = scores - s["slopes"][:, None] * (s["lens"][:, None, None] - 1 - key)
    live = live[:, None]
    scores = torch.where(live, scores, float("-inf"))
    most = scores.amax(dim=-1, keepdim=True)
    p = torch.where(live, torch.exp(scores - most), 0.0)
    total = p.sum(dim=-1, keepdim=True)
    v = torch.where(live[..., None], v, 0.0)
    out = torch.matmul(p.view(r, kvh, h // kvh, -1), v).view(r, h, d)
    return torch.where(total > 0, out / total, 0.0).to(s["q"].dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from scoreperformer_amd import ops
        if op == "plan":
            return (s["table"],) + tuple(ops.paged_plan(s["lens"], s["new"], s["table"], s["free"], s["num_free"], s["page"], s["width"]))
        if op == "turnover":
            ops.paged_release(s["done"], s["lens"], s["table"], s["free"], s["num_free"], s["page"])
            slots, _, _ = ops.paged_plan(s["lens"], s["new"], s["table"], s["free"], s["num_free"], s["page"], s["width"], lens_out=s["lens"],
                                         num_free_out=s["num_free"])
            return s["table"], slots, s["lens"], s["num_free"], s["free"]
        if op == "append":
            ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"])
            return s["k_pages"], s["v_pages"]
        return ops.paged_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], slopes=s["slopes"])
    if op == "plan":
        return (s["table"],) + _plan(s)
    if op == "turnover":
        _release(s)
        slots, lens, num_free = _plan(s)
        s["lens"].copy_(lens)
        s["num_free"].copy_(num_free)
        return s["table"], slots, s["lens"], s["num_free"], s["free"]
    return _append(s) if op == "append" else _attn(s)


# ------------------------------------------------------------------------------------------------------------------------- floors

def work(case):
    cached, new = _lengths(case)
    n, page = case["requests"], case["page"]
    if case["op"] == "append":
        row = case["kv_heads"] * HEAD * 2 * (SIZE[case["rows"]] + SIZE[case["pages"]])
        return dict(bytes=sum(new) * row + 8 * n * case["width"], flops=0)
    if case["op"] == "attn":
        row = case["kv_heads"] * HEAD * 2 * SIZE[case["dtype"]]
        pages = sum(_pages_of(c, page) for c in cached)
        return dict(bytes=sum(cached) * row + 4 * pages + 4 * n + 2 * n * case["heads"] * HEAD * SIZE[case["dtype"]] + (4 * case["heads"] if case["alibi"] else 0),
                    flops=4 * sum(cached) * case["heads"] * HEAD)
    ended = sum(_pages_of(c, page) for c, m in zip(cached, new) if m) if case["op"] == "turnover" else 0
    taken = ended or sum(_pages_of(c + m, page) - _pages_of(c, page) for c, m in zip(cached, new))
    # lengths in and out, new counts in, slots out; a page taken: its id read and written; a page put back the same
    return dict(bytes=12 * n + 8 * n * case["width"] + 8 * taken + 8 * ended + 8 + (n if ended else 0), flops=0)


# --------------------------------------------------------------------------------------------------------- the definition, exactly

def _exact_plan(table, lens, new, stack, page, width, num_pages):
    """Request by request, with a Python list as the stack; `stack`'s end is its top.  A request is served whole or not at all, and once the pages
    asked for so far are more than there are, nobody behind gets any."""
    asked, had = 0, len(stack)
    slots = np.full((len(lens), width), -1, dtype=np.int64)
    for r in range(len(lens)):
        end = lens[r] + new[r]
        if not 0 <= new[r] <= width or lens[r] < 0 or _pages_of(end, page) > table.shape[1]:
            continue
        need = _pages_of(end, page) - _pages_of(lens[r], page)
        asked += need
        if need and asked > had:
            continue
        for j in range(need):
            table[r, _pages_of(lens[r], page) + j] = stack.pop()
        pos = np.arange(lens[r], end)
        ids = table[r, pos // page].astype(np.int64)
        slots[r, :new[r]] = np.where((ids >= 0) & (ids < num_pages), ids * page + pos % page, -1)
        lens[r] = end
    return slots


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("plan", "turnover"):
        table, lens, new, free = (s[k].cpu().numpy().copy() for k in ("table", "lens", "new", "free"))
        lens, new = [int(x) for x in lens], [int(x) for x in new]
        stack = [int(x) for x in free[:int(s["num_free"])]]
        if case["op"] == "turnover":
            for r in reversed(np.nonzero(s["done"].cpu().numpy())[0]):
                for j in reversed(range(_pages_of(lens[r], case["page"]))):
                    stack.append(int(table[r, j]))
                    table[r, j] = -1
                lens[r] = 0
            free[:len(stack)] = stack
        slots = _exact_plan(table, lens, new, stack, case["page"], s["width"], len(free))
        got = [torch.from_numpy(x) for x in (table, slots, np.asarray(lens, dtype=np.int32), np.asarray([len(stack)], dtype=np.int32))]
        return tuple(got) + ((torch.from_numpy(free),) if case["op"] == "turnover" else ())
    if case["op"] == "append":
        slots = s["slots"].flatten().cpu()
        rows = torch.nonzero(slots >= 0)[:, 0]
        to = slots[rows]
        pools = []
        for new, pool in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
            flat = pool.double().transpose(1, 2).reshape(-1, pool.shape[1], HEAD)      # [slot, head, 64]
            flat.index_copy_(0, to.to(flat.device), new.double()[rows.to(flat.device)])
            pools.append(flat.view(pool.shape[0], pool.shape[2], pool.shape[1], HEAD).transpose(1, 2).contiguous())
        return tuple(pools)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group = case["heads"] // case["kv_heads"]
    for r, n in enumerate(s["lens"].tolist()):
        if not n:
            continue
        ids = s["table"][r, :_pages_of(n, case["page"])].long()
        k, v = (pool.index_select(0, ids).double().transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(group, dim=0) for pool in (s["k_pages"], s["v_pages"]))
        score = (k * s["q"][r].double()[:, None, :]).sum(-1) / math.sqrt(HEAD)
        if s["slopes"] is not None:
            score = score + s["slopes"].double()[:, None] * torch.arange(1 - n, 1, device=score.device, dtype=torch.float64)
        weight = torch.softmax(score, dim=-1)
        out[r] = (weight[:, :, None] * v).sum(1)
    return out
