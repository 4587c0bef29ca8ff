"""GPU: the paged attention over the longest table rows that a call accepts (2^31 less one page), nearly all of them holes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype, page", [(BF16, 8), (BF16, 16), (F32, 8)])
def test_attention_of_a_table_row_that_fills_the_range(dev, dtype, page):
    """Lengths whose last tile ends at row 2^31: the rows of the few pages there are, the newest one among them, far and near, with their bias.

    Tolerance: a score and its bias are off by at most ds = (68 + 4) u of their size (u = 2^-24; the distance itself is rounded to 32 bits), a
    probability by e^(2 ds), the exponential by 2^-21, the few sums by 16 u, all relative to the largest |v|; bf16 adds 2^-16 of the two-part
    probabilities and one rounding of the output, 2^-8 of it."""
    from scoreperformer_amd import ops
    W = 2 ** 31 // page - 1
    n = W * page
    at = [0, 1, W // 3, W // 2 + 1, W - 3, W - 1]                      # entries that are pages
    g = torch.Generator().manual_seed(page)
    kp, vp = (torch.randn(len(at) + 1, 2, page, 64, generator=g).to(dtype) for _ in range(2))     # (page 0: of nobody)
    table = torch.full((1, W), -1, device=dev, dtype=torch.int32)
    for i, j in enumerate(at):
        table[0, j] = i + 1
    q = torch.randn(1, 4, 64, generator=g).to(dtype)
    slopes = torch.tensor([0.0, 2.0 ** -31, 2.0 ** -30, 0.5])          # none; a bias of -1 and -2 at the first row; only the newest rows count
    for lens in (n, n - 1, n - page + 1):
        got = ops.paged_attn(q.to(dev), kp.to(dev), vp.to(dev), table, torch.tensor([lens], device=dev, dtype=torch.int32), slopes=slopes.to(dev)).cpu().double()
        pos = torch.cat([torch.arange(page) + j * page for j in at])
        live = pos < lens
        k, v = (p[1:].double().transpose(0, 1).flatten(1, 2)[:, live] for p in (kp, vp))          # [kvh, rows, 64]
        for h in range(4):
            qk = k[h // 2] * q[0, h].double() / 8
            s = qk.sum(-1) - slopes[h].double() * (lens - 1 - pos[live]).double()
            want = torch.softmax(s, 0) @ v[h // 2]
            u = 2.0 ** -24
            ds = 72 * u * (float(qk.abs().sum(-1).max()) + 50.0)       # (a bias beyond 50 leaves a weight below e^-30)
            tol = float(v.abs().max()) * (2 * ds + 2.0 ** -21 + 16 * u + (2.0 ** -16 if dtype is BF16 else 0)) + want.abs() * (2.0 ** -8 if dtype is BF16 else 2 * u)
            assert bool(((got[0, h] - want).abs() <= tol).all()), (lens, h, float(((got[0, h] - want).abs() / tol).max()))
