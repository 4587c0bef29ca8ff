"""GPU: the gradients of the embedding norm's gain and bias (spn_embed_bwd_det) are the same bits every time, at every number of notes.

Tolerance: with the kernel's own fp32 mean and rstd a term dy * xhat carries three roundings, and a column's sum goes through a known chain of adds
(rows of a wave, 4 waves, every 32nd block, 32 groups, the add into the gradient), each off by at most u = 2^-24 of what it has summed so far, so of
the sum of the absolute terms: (3 + chain) u sum |dy xhat|, plus one rounding of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
WIDTHS = {"12 x 128": [128] * 12, "4 x 128": [128] * 4, "5 x 32": [32] * 5, "odd": [36, 4, 100]}


def _case(dev, E, T, seed=0):
    from scoreperformer_amd import ops
    g = torch.Generator().manual_seed(seed + T)
    tables = [torch.randn(40 + i, e, generator=g).to(dev) for i, e in enumerate(E)]
    tokens = torch.stack([torch.randint(0, 40 + i, (1, T), generator=g) for i in range(len(E))], -1).to(dev)
    gamma, beta = (torch.rand(sum(E), generator=g).to(dev) + 0.5 for _ in range(2))
    _, mean, rstd = ops.embed_fwd(tables, tokens, gamma, beta)
    dy = torch.randn(T, sum(E), generator=g)
    dy[T // 2:2 * (T // 2)] = -dy[:T // 2]        # bias gradients of nothing but cancelling terms
    return tables, tokens, dy.to(dev).bfloat16(), gamma, mean, rstd


def _run(case, start=None):
    from scoreperformer_amd import ops
    dgamma, dbeta = (torch.zeros_like(case[3]) if start is None else start.clone() for _ in range(2))
    ops.embed_bwd(*case, dgamma=dgamma, dbeta=dbeta)
    return dgamma, dbeta


def _chain(T, blocks=2048):
    rows = (-(-T // blocks) + 3) // 4 * 4
    return rows // 4 + 4 + -(-T // rows) // 32 + 1 + 32 + 1


def _check(case, got, chain, start=0.0):
    tables, tokens, dy, _, mean, rstd = case
    x = torch.cat([t[tokens[0, :, k]] for k, t in enumerate(tables)], 1).double()
    d = dy.double()
    xh = (x - mean.double()[:, None]) * rstd.double()[:, None]
    for g, terms in ((got[0], d * xh), (got[1], d)):
        want = terms.sum(0) + start
        tol = (3 + chain) * U * (terms.abs().sum(0) + abs(start)) + U * want.abs()
        assert bool(((g.double() - want).abs() <= tol).all()), float(((g.double() - want).abs() / tol).max())


@pytest.mark.parametrize("T", [1, 4, 5, 127, 128, 129, 666, 4097, 20001])
@pytest.mark.parametrize("widths", list(WIDTHS))
def test_norm_gradients_are_the_same_every_time(dev, widths, T):
    case = _case(dev, WIDTHS[widths], T)
    first = _run(case)
    _check(case, first, _chain(T))
    for _ in range(6):
        again = _run(case)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    _check(case, _run(case, torch.full_like(first[0], 3.0)), _chain(T), 3.0)          # accumulates


@pytest.mark.parametrize("blocks", [1, 7, 100])
def test_norm_gradients_at_other_grids(dev, blocks):
    from scoreperformer_amd import lib
    case = _case(dev, WIDTHS["5 x 32"], 1000)
    old = lib.get_tuning("embed_stats_blocks")
    lib.set_tuning("embed_stats_blocks", blocks)
    try:
        first = _run(case)
        _check(case, first, _chain(1000, blocks))
        assert all(torch.equal(first[0], _run(case)[0]) for _ in range(4))
    finally:
        lib.set_tuning("embed_stats_blocks", old)


def test_norm_gradients_in_a_replayed_graph(dev):
    """Replays with eager work between them, on other gradients each time."""
    from scoreperformer_amd import ops
    case = _case(dev, WIDTHS["4 x 128"], 700)
    dy = case[2]
    dgamma, dbeta = (torch.zeros_like(case[3]) for _ in range(2))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.embed_bwd(*case, dgamma=dgamma, dbeta=dbeta)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dgamma.zero_()
        dbeta.zero_()
        ops.embed_bwd(*case, dgamma=dgamma, dbeta=dbeta)
    for it in range(6):
        dy.copy_(torch.randn(dy.shape, device=dev))
        g.replay()
        want = _run(case)
        if it % 2:
            torch.cuda.synchronize()
        assert torch.equal(dgamma, want[0]) and torch.equal(dbeta, want[1]), it


def test_the_form_without_a_larger_workspace_sums_the_same_terms(dev):
    """spn_embed_bwd, whose blocks add by atomics: the order is free, the terms are not."""
    from scoreperformer_amd import ops
    from scoreperformer_amd.lib import c_int, c_long, call, ptr, stream_ptr
    case = tables, tokens, dy, gamma, mean, rstd = _case(dev, WIDTHS["5 x 32"], 666)
    V, E = [t.shape[0] for t in tables], [t.shape[1] for t in tables]
    dts = [torch.zeros_like(t) for t in tables]
    dgamma, dbeta = (torch.zeros_like(gamma) for _ in range(2))
    ws = torch.empty(2 * 666, device=dev)
    call("spn_embed_bwd", c_int(len(E)), ops._ptr_array(tables), ops._ptr_array(dts), ops._int_array(V), ops._int_array(E), ptr(tokens),
         c_long(tokens.stride(0)), c_long(tokens.stride(1)), c_int(666), ptr(dy), c_long(dy.stride(0)), ptr(gamma), ptr(mean), ptr(rstd), ptr(dgamma),
         ptr(dbeta), ptr(ws), c_int(666), c_int(0), stream_ptr())
    _check(case, (dgamma, dbeta), 4 + 167)
