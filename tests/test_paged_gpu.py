"""GPU: the paged key / value cache (ops.paged_plan / paged_release / paged_append / paged_attn) against oracle/paged_cpu.py.

Whole numbers are equal.  Tolerance of the attention, from the arithmetic (fp32 u = 2^-24, d = 64): a score's products and bias are off by at
most ds = 68 u scale sum_i |q_i k_i| + 4 u (|s| + slope dist), so a probability by a factor e^(2 ds) and the exponential's own 2^-21; the sums
over n rows add independent roundings, 8 sqrt(n) u as a bound of eight standard deviations; all of it relative to the largest |v|.  bf16: a
probability that enters the matrix product in two bf16 parts keeps 2^-16 of itself, and the output is rounded once (2^-8)."""
import numpy as np
import pytest
import torch

from oracle import paged_cpu

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _ops():
    from scoreperformer_amd import ops
    return ops


def up(a, dev, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a)).to(device=dev, dtype=dtype)


# ----------------------------------------------------------------------------------------------------------------- plan and release

def _state(rng, R, W, page, num_pages, longest):
    lens = rng.integers(0, longest + 1, R).astype(np.int32)
    lens[rng.integers(0, R)] = 0
    lens[rng.integers(0, R)] = min(longest, page)
    held = -(-lens.astype(np.int64) // page)
    ids = rng.permutation(num_pages).astype(np.int32)
    table = np.full((R, W), -1, dtype=np.int32)
    table[np.arange(W)[None] < held[:, None]] = ids[:held.sum()]
    stack = np.full(num_pages, -7, dtype=np.int32)
    stack[:num_pages - held.sum()] = ids[held.sum():]
    return lens, table, stack, int(num_pages - held.sum())


def _run_plan(dev, lens, new, table, stack, free, page, width, inplace):
    ops = _ops()
    d_lens, d_new, d_table, d_stack, d_free = (up(x, dev) for x in (lens, new, table, stack, [free]))
    kw = dict(lens_out=d_lens, num_free_out=d_free) if inplace else {}
    slots, lens_out, free_out = ops.paged_plan(d_lens, d_new, d_table, d_stack, d_free, page, width, **kw)
    if not inplace:
        assert (d_lens.cpu().numpy() == lens).all() and int(d_free) == free
    assert (d_stack.cpu().numpy() == stack).all()
    want_table = table.copy()
    want = paged_cpu.plan([int(x) for x in lens], new, want_table, [int(x) for x in stack], free, page, width)
    assert slots.shape == (len(lens), width) and slots.dtype == torch.int64
    assert (slots.cpu().numpy() == want[0]).all()
    assert (lens_out.cpu().numpy() == want[1]).all() and int(free_out) == want[2]
    assert (d_table.cpu().numpy() == want_table).all()


@pytest.mark.parametrize("R, width, page", [(1, 1, 8), (1, 300, 16), (2, 7, 4096), (63, 1, 16), (64, 1, 16), (65, 33, 8), (300, 130, 32), (1023, 1, 8),
                                            (1024, 2, 16), (1025, 1, 16), (2500, 3, 8), (37, 1024, 64)])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan_matches_the_oracle(dev, R, width, page, inplace):
    rng = np.random.default_rng(R * 1000 + width)
    longest = 5 * page
    W = -(-(longest + width) // page)
    lens, table, stack, free = _state(rng, R, W, page, R * W + 3, longest)
    new = rng.integers(0, width + 1, R)
    new[rng.integers(0, R)] = width
    _run_plan(dev, lens, new, table, stack, free, page, width, inplace)


@pytest.mark.parametrize("R, width", [(40, 20), (1500, 20), (40, 700)])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan_refuses_requests_whole(dev, R, width, inplace):
    """Pages run out half way, counts outside [0, width], negative lengths, table rows too short, ids that are no pages."""
    rng = np.random.default_rng(5)
    page, W = 8, 6 + width // 8
    lens, table, stack, free = _state(rng, R, W, page, R * 4, 30)
    lens = lens.astype(np.int64)
    table = np.where(rng.random(table.shape) < 0.1, rng.choice([-1, -5, R * 4, 2 ** 31 - 1, -2 ** 31], table.shape), table).astype(np.int32)
    stack = np.where(rng.random(stack.shape) < 0.1, -3, stack).astype(np.int32)
    new = rng.integers(0, width + 1, R)
    for i, (l, n) in enumerate([(-1, 1), (5, -1), (3, width + 1), (2 ** 31 - 1, 1), (2 ** 31 - 2, width), (-2 ** 31, 0), (0, 2 ** 31 - 1), (W * 8, 1), (W * 8, 0)]):
        lens[3 + i], new[3 + i] = l, n
    _run_plan(dev, lens.astype(np.int32), new, table, stack, free, page, width, inplace)


@pytest.mark.parametrize("num_free", [0, -4, 10 ** 6])
def test_plan_with_a_bad_count_of_free_pages(dev, num_free):
    stack = np.arange(6, dtype=np.int32)
    _run_plan(dev, np.array([0, 8], np.int32), np.array([9, 9]), np.full((2, 4), -1, np.int32), stack, num_free, 8, 9, False)


def test_plan_of_no_request_and_a_table_slice(dev):
    ops = _ops()
    e = torch.zeros(0, device=dev, dtype=torch.int32)
    slots, lens, free = ops.paged_plan(e, e, torch.zeros(0, 3, device=dev, dtype=torch.int32), up([1, 2], dev), up([2], dev), 8, 4)
    assert slots.shape == (0, 4) and lens.shape == (0,) and int(free) == 2
    wide = torch.full((3, 10), -9, device=dev, dtype=torch.int32)      # columns 2 .. 5 of a wider table
    slots, lens, free = ops.paged_plan(up([0, 0, 0], dev), up([9, 0, 17], dev), wide[:, 2:6], up(range(7), dev), up([7], dev), 8, 17)
    want = np.full((3, 10), -9); want[0, 2:4] = [6, 5]; want[2, 2:5] = [4, 3, 2]
    assert (wide.cpu().numpy() == want).all() and int(free) == 2


@pytest.mark.parametrize("R, W, page", [(1, 1, 8), (5, 70, 8), (510, 64, 16), (1024, 3, 32), (1030, 9, 8), (2100, 130, 8)])
def test_release_matches_the_oracle_and_plan_undoes_it(dev, R, W, page):
    ops = _ops()
    rng = np.random.default_rng(R)
    lens, table, stack, free = _state(rng, R, W, page, R * W + 1, W * page)
    done = rng.random(R) < 0.5
    done[0] = True
    d = [up(done, dev, torch.bool)] + [up(x, dev) for x in (lens, table, stack, [free])]
    ops.paged_release(*d, page)
    w_lens, w_table, w_stack = lens.copy(), table.copy(), [int(x) for x in stack]
    w_free = paged_cpu.release(done, w_lens, w_table, w_stack, free, page)
    assert int(d[4]) == w_free
    for got, want in ((d[1], w_lens), (d[2], w_table), (d[3], w_stack)):
        assert (got.cpu().numpy() == np.asarray(want)).all()
    ops.paged_release(*d, page)                                      # ended requests hold nothing: nothing changes
    assert int(d[4]) == w_free and (d[3].cpu().numpy() == np.asarray(w_stack)).all()
    width = max(1, int(lens.max()))
    ops.paged_plan(d[1], up(np.where(done, lens, 0), dev), d[2], d[3], d[4], page, width, lens_out=d[1], num_free_out=d[4])
    assert (d[1].cpu().numpy() == lens).all() and (d[2].cpu().numpy() == table).all() and int(d[4]) == free


def test_release_of_broken_state_stays_in_bounds(dev):
    """Ids that are no pages, lengths past the table, a page held twice (more pages come back than there are)."""
    ops = _ops()
    lens = np.array([24, 2 ** 31 - 1, -5, 40], dtype=np.int32)
    table = np.array([[0, -1, 9], [1, 2, 2 ** 31 - 1], [3, 4, 5], [1, 2, 3]], dtype=np.int32)
    stack = np.array([4, 5, -9, -9, -9, -9], dtype=np.int32)
    done = np.array([1, 1, 1, 1], dtype=bool)
    d = [up(done, dev, torch.bool)] + [up(x, dev) for x in (lens, table, stack, [2])]
    ops.paged_release(*d, 8)
    w_stack = [int(x) for x in stack]
    w_free = paged_cpu.release(done, lens, table, w_stack, 2, 8)
    assert w_free == 6 and int(d[4]) == 6 and (d[3].cpu().numpy() == w_stack).all()
    assert (d[2].cpu().numpy() == table).all() and (d[1].cpu().numpy() == 0).all()


# ----------------------------------------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("rows", [BF16, F32])
@pytest.mark.parametrize("pages", [BF16, F32])
@pytest.mark.parametrize("T, kvh, page, skew", [(1, 1, 16, 0), (64, 1, 16, 0), (65, 3, 8, 0), (333, 8, 64, 0), (130, 2, 16, 1), (57, 1, 32, 4)])
def test_append_matches_the_oracle(dev, rows, pages, T, kvh, page, skew):
    """Rows read in place out of a fused buffer (skew: element offset of the slice, so that rows are not 16-byte aligned); slots that are none are
    skipped and nothing else of the pool is touched."""
    ops = _ops()
    rng = np.random.default_rng(T)
    n = -(-T // page) + 3
    slots = rng.permutation(n * page)[:T].astype(np.int64)
    bad = rng.random(T) < 0.2
    slots[bad] = rng.choice([-1, -100, n * page, n * page + 5, 2 ** 40, -2 ** 62], bad.sum())
    g = torch.Generator().manual_seed(T)
    fused = torch.randn(T, 64 + 2 * kvh * 64 + 8, generator=g).to(rows).to(dev)
    k, v = (fused[:, 64 + skew + i * kvh * 64:64 + skew + (i + 1) * kvh * 64].unflatten(1, (kvh, 64)) for i in (0, 1))
    pools = [torch.randn(n, kvh, page, 64, generator=g).to(pages) for _ in range(2)]
    got = [p.to(dev) for p in pools]
    ops.paged_append(k, v, got[0], got[1], up(slots, dev, torch.int64).view(1, T))
    for p, r, x in ((pools[0], k, got[0]), (pools[1], v, got[1])):
        paged_cpu.append(r.cpu(), p, torch.from_numpy(slots))
        assert torch.equal(x.cpu().view(torch.uint8), p.view(torch.uint8))       # bit for bit


def test_append_keeps_infinities_and_nan_and_head_strides(dev):
    ops = _ops()
    src = torch.randn(2, 40, 64, device=dev)                      # [head, row, 64]: head-major rows
    src[0, 0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    src[1, 5, 0] = 3.4e38                                         # rounds to infinity in bf16
    kp, vp = (torch.zeros(6, 2, 8, 64, device=dev, dtype=BF16) for _ in range(2))
    slots = torch.arange(40, device=dev)
    ops.paged_append(src.transpose(0, 1), (-src).transpose(0, 1), kp, vp, slots)
    want = src.to(BF16)
    back = kp.transpose(0, 1).flatten(1, 2)[:, :40]
    assert torch.equal(torch.nan_to_num(back, nan=123.0), torch.nan_to_num(want, nan=123.0)) and bool(back[0, 0, 2].isnan())
    assert torch.equal(torch.nan_to_num(vp.transpose(0, 1).flatten(1, 2)[:, :40], nan=123.0), torch.nan_to_num(-want, nan=123.0))
    ops.paged_append(src[:, :0].transpose(0, 1), src[:, :0].transpose(0, 1), kp, vp, slots[:0])


# -------------------------------------------------------------------------------------------------------------------------- attention

def _cache(dev, lens, kvh, page, dtype, seed=0, W=None, extra=3, poison=float("nan")):
    """Random pages in random order; rows that no request holds are `poison`."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    held = -(-lens // page)
    W = max(1, int(held.max())) if W is None else W
    n = int(held.sum()) + extra
    ids = rng.permutation(n)
    table = np.full((len(lens), W), -1, dtype=np.int64)
    table[np.arange(W)[None] < held[:, None]] = ids[:held.sum()]
    kp, vp = (torch.full((n, kvh, page, 64), poison).to(dtype) for _ in range(2))
    for r, m in enumerate(lens):
        for j in range(0, int(m), page):
            c = min(page, int(m) - j)
            for p in (kp, vp):
                p[table[r, j // page], :, :c] = torch.randn(kvh, c, 64, generator=g).to(dtype)
    return kp, vp, torch.from_numpy(table).int(), torch.as_tensor(lens).int()


def _slopes(h):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)])


def _tolerance(q, kp, vp, table, lens, slopes, scale, want):
    n = max(1, int(lens.max()))
    page = kp.shape[2]
    finite = torch.nan_to_num(kp.double(), nan=0.0, posinf=0.0, neginf=0.0)
    s_abs = float(scale * q.double().abs().max(1)[0].max(0)[0] @ finite.abs().amax(dim=(0, 1, 2)))
    reach = float(slopes.max()) * n if slopes is not None else 0.0
    # a bias so large that its rounding matters belongs to a row of weight exp(-bias): only the part up to 100 counts
    ds = 68 * U * s_abs + 4 * U * (s_abs + min(reach, 100.0 + 2 * s_abs))
    vmax = float(torch.nan_to_num(vp.double(), nan=0.0, posinf=0.0, neginf=0.0).abs().max())
    rel = 2 * ds + 2.0 ** -21 + 8 * n ** 0.5 * U
    if q.dtype == BF16:
        return vmax * (rel + 2.0 ** -16) + want.abs() * 2.0 ** -8
    return vmax * rel + want.abs() * 2 * U


def _check(dev, q, kp, vp, table, lens, slopes=None, scale=None, **kw):
    got = _ops().paged_attn(q.to(dev) if not q.is_cuda else q, kp.to(dev), vp.to(dev), table.to(dev), lens.to(dev),
                            slopes=None if slopes is None else slopes.to(dev), scale=scale, **kw)
    want = paged_cpu.attn(q.cpu(), kp, vp, table, lens, scale, slopes)
    assert got.shape == q.shape and got.dtype == q.dtype
    off = (got.cpu().double() - want).abs()
    tol = _tolerance(q.cpu(), kp, vp, table, lens, slopes, 0.125 if scale is None else scale, want)
    assert bool((off <= tol).all()), (float(off.max()), float((off / tol).max()))
    return got


LENS = {"one": [1], "none": [0], "tile-edges": [0, 1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129], "long": [1000, 0, 1537, 3],
        "many": [(i * 37) % 301 for i in range(150)], "single-long": [5003]}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(8, 1), (1, 1), (6, 3), (8, 8), (20, 1), (40, 2)])
@pytest.mark.parametrize("which", list(LENS))
@pytest.mark.parametrize("page, bias", [(16, True), (8, False), (128, True)])
def test_attention_matches_the_oracle(dev, dtype, heads, which, page, bias):
    h, kvh = heads
    lens = LENS[which]
    kp, vp, table, lens = _cache(dev, lens, kvh, page, dtype, seed=h)
    q = torch.randn(len(lens), h, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    got = _check(dev, q, kp, vp, table, lens, _slopes(h) if bias else None)
    assert bool((got[(lens == 0).to(dev)] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kvh, lens, page", [(8, [(i * 53) % 901 for i in range(40)], 16),           # whole segments: 4 waves each
                                             (8, [(i * 311) % 2101 for i in range(33)], 8),           # 8 waves, long tables
                                             (8, [4096 - (i * 331) % 4096 for i in range(36)], 64),    # 8 waves, rows not kept in the caches
                                             (1, [70001], 32), (1, [131, 40000, 7], 16),               # cut: many parts of one request
                                             (4, [20000, 0, 39999, 25000], 128)])                      # cut, rows not kept in the caches
def test_attention_of_large_batches_matches_the_oracle(dev, dtype, kvh, lens, page):
    """The sizes at which the work is divided and the rows are read in other ways."""
    kp, vp, table, lens = _cache(dev, lens, kvh, page, dtype, seed=7)
    q = torch.randn(len(lens), 8, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    _check(dev, q, kp, vp, table, lens, _slopes(8) / 64)      # shallow slopes: far rows count


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("heads", [(8, 8), (20, 1)])
@pytest.mark.parametrize("longest, wide", [(120, 0), (120, 20000), (1700, 0), (1700, 20000), (6000, 0)])
def test_attention_of_thousands_of_segments(dev, dtype, page, heads, longest, wide):
    """More requests x key heads than run at once: short ones a wave each, long ones among them, in narrow tables and in tables far wider than any
    length (other ways of dividing the work: the result is the same)."""
    h, kvh = heads
    R = 2063 // kvh if kvh > 1 else 1031
    lens = [(i * 37) % 121 for i in range(R)]
    lens[5], lens[R - 1], lens[R // 2] = longest, longest - 3, 0
    kp, vp, table, lens = _cache(dev, lens, kvh, page, dtype, seed=page)
    if wide:
        table = torch.cat([table, torch.full((R, wide // page - table.shape[1]), -1, dtype=torch.int32)], 1)
    _check(dev, torch.randn(R, h, 64, generator=torch.Generator().manual_seed(3)).to(dtype), kp, vp, table, lens, _slopes(h) / 8)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R, h, kvh", [(256, 2, 1), (257, 2, 1), (512, 2, 1), (1025, 34, 2), (4097, 2, 2), (9000, 1, 1)])
def test_attention_of_thousands_of_requests_in_wide_tables(dev, dtype, R, h, kvh):
    """The line of parts over more requests than a wave, a workgroup, 64 x 64 searches hold; cut requests first, last and in between."""
    lens = [(i * 29) % 41 for i in range(R)]
    for i, n in ((0, 5000), (R - 1, 900), (R // 2, 2500), (63, 700), (64, 701)):
        lens[i] = n
    kp, vp, table, lens = _cache(dev, lens, kvh, 16, dtype, seed=R)
    table = torch.cat([table, torch.full((R, 1300 - table.shape[1]), -1, dtype=torch.int32)], 1)
    _check(dev, torch.randn(R, h, 64, generator=torch.Generator().manual_seed(4)).to(dtype), kp, vp, table, lens, _slopes(h) / 8)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, 1e-30, -0.125, 1e-12, 3.0])
def test_attention_with_any_scale(dev, dtype, scale):
    kp, vp, table, lens = _cache(dev, [300, 5, 0], 2, 8, dtype)
    q = torch.randn(3, 6, 64).to(dtype)
    got = _ops().paged_attn(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), lens.to(dev), scale=scale, slopes=_slopes(6).to(dev))
    want = paged_cpu.attn(q, kp, vp, table, lens, scale, _slopes(6))
    assert bool(((got.cpu().double() - want).abs() <= _tolerance(q, kp, vp, table, lens, _slopes(6), abs(scale), want)).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_in_place_of_its_query_and_over_a_slice_of_a_wider_table(dev, dtype):
    kp, vp, table, lens = _cache(dev, [700, 31, 0, 2500], 2, 16, dtype)
    wide = torch.full((4, table.shape[1] + 9), 2 ** 31 - 1, dtype=torch.int32)
    wide[:, 4:4 + table.shape[1]] = table
    q = torch.randn(4, 4, 64).to(dtype)
    want = _ops().paged_attn(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), lens.to(dev))
    d_q = q.to(dev)
    got = _ops().paged_attn(d_q, kp.to(dev), vp.to(dev), wide.to(dev)[:, 4:4 + table.shape[1]], lens.to(dev), out=d_q)
    assert got is d_q and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_strides_scale_and_given_output(dev, dtype):
    """q as a slice of the fused projection, heads in front; the output into a slice of a wider buffer, nothing beside it touched."""
    kp, vp, table, lens = _cache(dev, [40, 3, 77], 2, 16, dtype)
    fused = torch.randn(3, 4 * 64 + 24).to(dtype).to(dev)
    _check(dev, fused[:, 3:3 + 256].unflatten(1, (4, 64)), kp, vp, table, lens, _slopes(4), scale=0.3)
    _check(dev, torch.randn(4, 3, 64).to(dtype).to(dev).transpose(0, 1), kp, vp, table, lens)
    out = torch.full((3, 7, 64 + 5), 7.0, device=dev, dtype=dtype)
    q = torch.randn(3, 4, 64).to(dtype).to(dev)
    got = _check(dev, q, kp, vp, table, lens, out=out[:, 2:6, 3:67])
    assert got.data_ptr() == out[:, 2:6, 3:67].data_ptr()
    out[:, 2:6, 3:67] = 7.0
    assert bool((out == 7).all())
    _check(dev, q, kp, vp, table, lens, out=torch.empty(4, 3, 64, device=dev, dtype=dtype).transpose(0, 1))      # heads in front


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [8, 16, 64])
def test_attention_skips_what_is_no_page_and_cuts_long_lengths(dev, dtype, page):
    kp, vp, table, lens = _cache(dev, [400, 390, 64, 64, 300], 1, page, dtype)
    rng = np.random.default_rng(3)
    holes = torch.from_numpy(rng.random(table.shape) < 0.3)
    holes[2] = True                                               # a request without a page: zeros
    holes[3, :], holes[3, 0] = True, False                        # only its first page
    bad = torch.from_numpy(rng.choice([-1, -2 ** 31, kp.shape[0], 2 ** 31 - 1], table.shape)).int()
    table = torch.where(holes, bad, table)
    lens[1], lens[4] = table.shape[1] * page + 123, -7            # past the table's pages; negative: nothing
    if page * table.shape[1] > 390:
        kp, vp = (torch.nan_to_num(p, nan=0.5) for p in (kp, vp))  # the cut length reaches rows that nobody wrote
    q = torch.randn(5, 8, 64).to(dtype)
    got = _check(dev, q, kp, vp, table, lens, _slopes(8))
    assert bool((got[2] == 0).all()) and bool((got[4] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_large_scores_and_one_dominant_row(dev, dtype):
    """Scores of thousands of either sign (the softmax is taken relative to the maximum), a maximum that moves at every row, and a row that alone
    carries the result: its value comes back, wherever it lies."""
    n = 300
    kp, vp, table, lens = _cache(dev, [n], 1, 16, F32, poison=0.0)
    for at in (0, 1, 31, 32, 150, n - 1):
        k = kp.clone()
        rows = [(int(table[0, j // 16]), j % 16) for j in range(n)]
        for j, (p, o) in enumerate(rows):
            k[p, 0, o] = -40.0 + 0.125 * (j % 64)
        k[rows[at][0], 0, rows[at][1]] = 40.0
        q = torch.full((1, 8, 64), 2.0)
        got = _ops().paged_attn(q.to(dtype).to(dev), k.to(dtype).to(dev), vp.to(dtype).to(dev), table.to(dev), lens.to(dev))
        want = vp.to(dtype)[rows[at][0], 0, rows[at][1]]
        assert torch.equal(got.cpu(), want.expand(1, 8, 64)), at
    k = kp.clone()
    for j in range(n):
        k[int(table[0, j // 16]), 0, j % 16] = 0.1 * j            # rising maximum
    _check(dev, torch.full((1, 8, 64), 0.5).to(dtype), k.to(dtype), vp.to(dtype), table, lens)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_keeps_numbers_that_are_none_to_their_own_head_and_request(dev, dtype):
    """A NaN among a request's visible keys of one key head gives that head NaN, and no other; a NaN value the same for its dimension."""
    kp, vp, table, lens = _cache(dev, [50, 50], 2, 16, dtype)
    clean = _ops().paged_attn(torch.ones(2, 4, 64, dtype=dtype, device=dev), kp.to(dev), vp.to(dev), table.to(dev), lens.to(dev))
    kp[int(table[0, 1]), 1, 3, 5] = float("nan")
    vp[int(table[1, 2]), 0, 0, 9] = float("nan")
    got = _ops().paged_attn(torch.ones(2, 4, 64, dtype=dtype, device=dev), kp.to(dev), vp.to(dev), table.to(dev), lens.to(dev))
    bad = torch.zeros(2, 4, 64, dtype=torch.bool)
    bad[0, 2:], bad[1, :2, 9] = True, True
    assert torch.equal(got.isnan().cpu(), bad)
    assert torch.equal(got.cpu()[~bad], clean.cpu()[~bad])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_a_pool_past_2_to_31_elements(dev, dtype):
    """Offsets in 64 bits: the pages in use are the last ones of a pool of more than 2^31 elements (4 to 8 GiB each)."""
    page, kvh = 64, 8
    n = 2 ** 31 // (page * kvh * 64) + 40
    kp, vp, table, lens = _cache(dev, [1000, 130], kvh, page, dtype, extra=0, poison=0.0)
    big = []
    for p in (kp, vp):
        b = torch.empty(n, kvh, page, 64, device=dev, dtype=dtype)
        b[n - p.shape[0]:] = p.to(dev)
        big.append(b)
    q = torch.randn(2, 8, 64).to(dtype)
    got = _ops().paged_attn(q.to(dev), big[0], big[1], torch.where(table >= 0, table + n - kp.shape[0], table).to(dev), lens.to(dev), slopes=_slopes(8).to(dev))
    want = _ops().paged_attn(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), lens.to(dev), slopes=_slopes(8).to(dev))
    assert torch.equal(got, want)
    rows = torch.randn(3, kvh, 64, device=dev).to(dtype)
    slots = torch.tensor([n * page - 1, (n - 1) * page, n * page - 7], device=dev)
    _ops().paged_append(rows, rows + 1, big[0], big[1], slots)
    for i, o in enumerate((63, 0, 57)):
        assert torch.equal(big[0][n - 1, :, o], rows[i]) and torch.equal(big[1][n - 1, :, o], (rows + 1)[i])


def test_attention_of_no_request(dev):
    kp = torch.zeros(2, 1, 8, 64, device=dev)
    out = _ops().paged_attn(torch.zeros(0, 8, 64, device=dev), kp, kp.clone(), torch.zeros(0, 3, device=dev, dtype=torch.int32),
                            torch.zeros(0, device=dev, dtype=torch.int32))
    assert out.shape == (0, 8, 64)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_is_the_same_every_time(dev, dtype):
    """No sum depends on the order in which workgroups finish."""
    kp, vp, table, lens = (x.to(dev) for x in _cache(dev, [3001, 17, 0, 900], 2, 16, dtype))
    q = torch.randn(4, 8, 64, device=dev).to(dtype)
    first = _ops().paged_attn(q, kp, vp, table, lens, slopes=_slopes(8).to(dev))
    for _ in range(5):
        assert torch.equal(_ops().paged_attn(q, kp, vp, table, lens, slopes=_slopes(8).to(dev)), first)


# ------------------------------------------------------------------------------------------------------------------ streams and graphs

def test_calls_on_two_streams_do_not_share_scratch(dev):
    """Two long calls in flight at once, each on a stream of its own, and their results as one after the other."""
    data = [[x.to(dev) for x in _cache(dev, [4000, 1200 + i, 9], 1, 16, BF16, seed=i)] for i in (1, 2)]
    q = torch.randn(3, 8, 64, device=dev).to(BF16)
    want = [_ops().paged_attn(q, *d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_ops().paged_attn(q, *data[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


def test_a_decode_step_captured_and_replayed(dev):
    """plan (in place) -> append -> attention in one graph: every replay takes the lengths, pages and rows that are there then, with eager work and
    synchronisation between the replays; two graphs over two caches replayed in turn."""
    ops = _ops()
    page, R, h, kvh, W, N = 8, 5, 8, 2, 6, 40
    rng = np.random.default_rng(0)

    class Cache:
        def __init__(self):
            self.lens, self.new = torch.zeros(R, device=dev, dtype=torch.int32), torch.zeros(R, device=dev, dtype=torch.int32)
            self.table = torch.full((R, W), -1, device=dev, dtype=torch.int32)
            self.stack, self.free = up(rng.permutation(N), dev), up([N], dev)
            self.kp, self.vp = (torch.full((N, kvh, page, 64), float("nan"), device=dev, dtype=BF16) for _ in range(2))
            self.qkv = torch.zeros(R, (h + 2 * kvh) * 64, device=dev, dtype=BF16)
            self.slopes = _slopes(h).to(dev)
            self.rows = [[] for _ in range(R)]

        def step(self):
            slots, _, _ = ops.paged_plan(self.lens, self.new, self.table, self.stack, self.free, page, 1, lens_out=self.lens, num_free_out=self.free)
            k, v = (self.qkv[:, (h + i * kvh) * 64:(h + (i + 1) * kvh) * 64].unflatten(1, (kvh, 64)) for i in (0, 1))
            ops.paged_append(k, v, self.kp, self.vp, slots)
            return ops.paged_attn(self.qkv[:, :h * 64].unflatten(1, (h, 64)), self.kp, self.vp, self.table, self.lens, slopes=self.slopes)

    caches = [Cache(), Cache()]
    for c in caches:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            c.step()
        s.synchronize()
        c.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(c.graph):
            c.out = c.step()
    for it in range(20):
        for c in caches:
            new = rng.integers(0, 2, R)
            c.new.copy_(up(new, dev))
            c.qkv.copy_(torch.randn(c.qkv.shape, device=dev))
            c.graph.replay()
            if it % 3 == 0:
                torch.cuda.synchronize()
            row = c.qkv.cpu()
            for r in range(R):
                if new[r]:
                    c.rows[r].append(row[r, h * 64:])
            assert c.lens.tolist() == [len(x) for x in c.rows]
            want = torch.zeros(R, h, 64, dtype=torch.float64)
            for r in range(R):
                if c.rows[r]:
                    n = len(c.rows[r])
                    kv = torch.stack(c.rows[r]).double().view(n, 2, kvh, 64).repeat_interleave(h // kvh, 2)
                    sc = torch.einsum("jhd,hd->hj", kv[:, 0], row[r, :h * 64].double().view(h, 64)) / 8 + _slopes(h).double()[:, None] * torch.arange(1 - n, 1).double()
                    want[r] = torch.einsum("hj,jhd->hd", torch.softmax(sc, 1), kv[:, 1])
            assert float((c.out.cpu().double() - want).abs().max()) <= 2.0 ** -8 * 5, it       # |o| <= max |v| < 5: one rounding of the output


@pytest.mark.parametrize("R", [3, 300])
def test_graphs_of_cut_batches_replayed_at_once(dev, R):
    """Captured calls in tables far wider than the lengths (cut segments, the line drawn by every wave / in front): each replay divides the lengths that
    are there then, and two graphs in flight on two streams have scratch of their own."""
    ops, rng = _ops(), np.random.default_rng(R)
    calls = []
    for seed in (1, 2):
        kp, vp, table, lens = _cache(dev, [2100] * 3 + [40] * (R - 3), 2, 16, BF16, seed=seed)
        table = torch.cat([table, torch.full((R, 1500), -1, dtype=torch.int32)], 1)
        d = [x.to(dev) for x in (torch.randn(R, 8, 64).to(BF16), kp, vp, table, lens)]
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            ops.paged_attn(*d)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.paged_attn(*d)
        calls.append((s, g, d, out))
    for it in range(8):
        for _, _, d, _ in calls:
            n = rng.integers(0, 41, R)
            n[:3] = rng.integers(0, 2101, 3)
            d[4].copy_(torch.from_numpy(n).int())
        torch.cuda.synchronize()
        for _ in range(3):
            for s, g, _, _ in calls:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for _, _, d, out in calls:
            assert torch.equal(out, ops.paged_attn(*d)), it
