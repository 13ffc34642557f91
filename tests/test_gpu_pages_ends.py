"""The paged cache at the ends of its ranges, on the GPU.

Roundings that the tolerances count (half a step each, relative): f32 2^-24, bf16 2^-8, f16 2^-11."""
import pytest
import torch
from test_gpu_pages import gen_of, ints, random_pool

pytestmark = pytest.mark.gpu

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
