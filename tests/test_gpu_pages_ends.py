"""The paged cache at the ends of its ranges, on the GPU.

Roundings that the tolerances count (half a step each, relative): f32 2^-24, bf16 2^-8, f16 2^-11."""
import pytest
import torch
from test_gpu_pages import BF16, attn64, gen_of, ints, random_pool

pytestmark = pytest.mark.gpu

WEIGHTS = 2.0 ** -10      # of sum p |v|: see test_gpu_pages.py
LAST = 2 ** 31 - 1      # the last position that a descriptor can name


# ---- positions near 2^31 --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("far", [[110, 50, LAST - 40, 0], [110, 50, LAST, 0], [-5, 15, LAST - 3, 0], [110, 50, LAST - 49, 0]], ids=str)
def test_append_behind_positions_that_wrap(far):
    """A descriptor whose positions pass 2^31 is not stored, and the sequences behind it in the list are."""
    pool = random_pool(gen_of(51), 1, 12, 2, 64, 16, [0, 70, 30])
    g = gen_of(52)
    x, q = torch.randn(160, 2, 64, generator=g, device="cuda"), torch.randn(160, 4, 64, generator=g, device="cuda")
    keep = [t.clone() for t in (pool.k, pool.v, pool.ks, pool.vs)]
    alone = random_pool(gen_of(51), 1, 12, 2, 64, 16, [0, 70, 30])
    rest = [[10, 70, 0, 1], [80, 30, 0, 2]]
    alone.append(0, None, None, x, -x, ints(rest))
    qo = torch.zeros_like(q)
    pool.append(0, None, q, x, -x, ints([far] + rest), qo)
    for a, b, was in zip((pool.k, pool.v, pool.ks, pool.vs), (alone.k, alone.v, alone.ks, alone.vs), keep):
        assert torch.equal(a, b) and not torch.equal(a, was)
    row = torch.arange(160, device="cuda")
    named = (row >= 10) & (row < 110) | (row >= far[0]) & (row < far[0] + far[1]) & (far[2] + row - far[0] <= LAST)      # positions that there are
    assert torch.equal(qo, torch.where(named[:, None, None], q, 0))


@pytest.mark.parametrize("rows", [1, 30])
@pytest.mark.parametrize("page", [16, 64])
def test_attn_at_positions_that_wrap(rows, page):
    """Rows whose positions lie beyond the table's row, up to 2^31 - 1 and past it, attend all that has a page, as far as the window reaches."""
    g = gen_of(53)
    pool = random_pool(g, 2, 30, 2, 64, page, [150, 90])
    q = torch.randn(3 * rows + 2, 8, 64, generator=g, device="cuda").to(torch.bfloat16)
    for pos in (LAST - rows + 1, LAST, LAST - rows // 2):
        seqs = [[0, rows, pos, 0], [rows, rows, 60, 1], [2 * rows, rows, 5000, 0]]
        want, size = attn64(pool, 1, q, [[0, rows, 100000, 0], seqs[1], seqs[2]], 0.125, 0)
        o = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device="cuda")
        pool.attn(1, q, ints(seqs), o, max_rows=rows)
        n = 3 * rows
        assert bool(((o.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size)[:n].all())
        assert bool((o[n:] == 5.0).all())
    # windows: all of int32's range, from before position 0 on, and one that ends before the last position does
    seqs = [[0, rows, -3, 0], [rows, rows, LAST - 200, 1], [2 * rows, rows, 40, 1]]
    o = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device="cuda")
    pool.attn(1, q, ints(seqs), o, max_rows=rows, window=LAST)
    want, size = attn64(pool, 1, q, [seqs[0], seqs[2]], 0.125, 0)
    far, fsize = attn64(pool, 1, q, [[rows, rows, 100000, 1]], 0.125, 0)      # windows that begin before position 0
    want, size = want + far, size + fsize
    assert bool(((o.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size)[:3 * rows].all())
    pool.attn(1, q, ints([[0, rows, LAST - rows + 1, 0]]), o, max_rows=rows, window=LAST - 60)      # keys from about 60 on
    want, size = torch.zeros_like(want), torch.zeros_like(size)
    for i in range(rows):
        lo = LAST - rows + 1 + i - (LAST - 60) + 1
        w, s = attn64(pool, 1, q, [[i, 1, 100000, 0]], 0.125, 100001 - lo)
        want, size = want + w, size + s
    assert bool(((o.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size)[:rows].all())
