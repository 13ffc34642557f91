"""The paged cache at the ends of its ranges, on the GPU.

Roundings that the tolerances count (half a step each, relative): f32 2^-24, bf16 2^-8, f16 2^-11."""
import math
import threading
from fractions import Fraction

import pytest
import torch
from test_gpu_pages import BF16, F32, P, attn64, check_attn, gen_of, held, ints, inv_of, random_pool, turned

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


# ---- angles of far positions ------------------------------------------------------------------------------------------------------
PI = Fraction(314159265358979323846264338327950288419716939937510582097494459230781640628620899, 10 ** 80)


@pytest.mark.parametrize("first", [-2 ** 31, 2 ** 29 + 1, 2 ** 30 + 3, LAST - 63])
def test_rope_angles_are_exact(first):
    """cos and sin of pos * inv, the product and its reduction to a quarter turn in exact fractions.  The result is rounded to f32 once (2^-24 of it); sums of Taylor
    terms up to r^11 and r^10 leave out at most (pi/4)^12 / 12! < 1.2e-10, and a few roundings in 64 bits, 1e-15."""
    vals = [1.0, 0.7310585786300049, 0.99999994, 1e-3, 0.5000001, 0.1234567, 3e-5, 0.9] + [10000.0 ** (-2 * p / 16) * 0.9876543 for p in range(8)]
    inv = torch.tensor(vals, dtype=torch.float32)
    pos = list(range(first, first + 64))
    x = torch.zeros(64, 1, 64, device="cuda")
    x[..., :16] = 1.0      # pairs (1, 0): the rotated pair is (cos, sin)
    P().rope(P().Rope(inv.cuda()), x, None, ints(pos))
    got = x.cpu().double()
    for t, p in enumerate(pos):
        for i in range(16):
            a = Fraction(p) * Fraction(float(inv[i]))
            k = round(a / (PI / 2))
            r = float(a - k * PI / 2)
            c, s = [(math.cos(r), math.sin(r)), (-math.sin(r), math.cos(r)), (-math.cos(r), -math.sin(r)), (math.sin(r), -math.cos(r))][k % 4]
            assert abs(float(got[t, 0, i]) - c) <= F32 * abs(c) + 1.3e-10, (p, i)
            assert abs(float(got[t, 0, i + 16]) - s) <= F32 * abs(s) + 1.3e-10, (p, i)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hd,rot,factor", [(64, 64, 1.0), (128, 64, 1.25), (256, 256, 1.0)])
def test_rope_rounds_each_step_once(hd, rot, factor, inter):
    """Sine and cosine times the factor, the two products and their sum: 3 roundings to f32 of factor (|u| + |w|) at most, and 1.2e-10 of it from the Taylor sums."""
    g = gen_of(55)
    x = torch.randn(500, 3, hd, generator=g, device="cuda")
    pos = torch.randint(0, 2 ** 29, (500,), generator=g, device="cuda", dtype=torch.int32)
    r = P().Rope(inv_of(rot), interleaved=inter, factor=factor)
    out = torch.empty_like(x)
    P().rope(r, x, None, pos, out)
    want, size = turned(x, pos, r.inv, inter, factor)
    assert bool(((out.double() - want).abs() <= 3.01 * F32 * factor * size).all())


# ---- lengths that are none ----------------------------------------------------------------------------------------------------------
def test_management_of_a_length_below_zero():
    """A sequence whose length the host has spoilt: its requests are refused, nobody else's page or entry changes."""
    pool = P().PagePool.empty(1, 40, 1, 64, 16, 3, 10)
    got = ints([7, 7, 7])
    pool.extend(ints([[0, 160], [1, 20], [2, 20]]), got)
    pool.length[1] = -100
    table, ref = pool.table.clone(), pool.ref.clone()
    pool.extend(ints([[1, 50], [2, 40], [0, 161]]), got)
    assert got.tolist() == [0, 1, 0]
    pool.trim(ints([[1, 0]]))
    pool.fork(ints([[1, 2, 5, 0]]))
    assert pool.length.tolist() == [160, -100, 40]
    table[2, 2] = pool.table[2, 2]
    ref[pool.table[2, 2]] = 1
    assert torch.equal(pool.table, table) and torch.equal(pool.ref, ref)
    pool.length[1] = 2 ** 31 - 1
    pool.extend(ints([[1, 50], [2, 5], [0, 3]]), got)
    assert got.tolist() == [0, 1, 1] and torch.equal(pool.table, table) and torch.equal(pool.ref, ref)


# ---- waits that run out -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,group,hd,page,code", [(1, 8, 128, 64, 2), (2, 4, 64, 16, 2), (3, 8, 64, 32, 7), (20, 2, 128, 128, 7), (200, 4, 128, 64, 7)], ids=str)
def test_attn_wait_that_runs_out(rows, group, hd, page, code):
    """Codes that are never fetched: every block's wait for them ends after its bound, the results are NaN and the status says why, rows that nobody
    names stay, and the next call is right."""
    lib = P().L.load()
    g = gen_of(56 + rows)
    lengths = [3000, 400, 70 + rows]
    pool = random_pool(g, 2, sum(-(-n // page) for n in lengths), 2, hd, page, lengths)
    q = torch.randn(3 * rows + 2, 2 * group, hd, generator=g, device="cuda").to(torch.bfloat16)
    seqs = [[i * rows, rows, n - rows, i] for i, n in enumerate(lengths)]
    check_attn(pool, q, seqs)
    assert pool.status() == 0
    o = torch.full_like(q, 5.0)
    lib.nsl_pages_attn_hold(3_000_000)      # ns
    try:
        pool.attn(1, q, ints(seqs), o, max_rows=rows)
        torch.cuda.synchronize()
    finally:
        lib.nsl_pages_attn_hold(0)
    assert bool(o[:3 * rows].isnan().all()) and bool((o[3 * rows:] == 5.0).all())
    got = pool.status()
    assert got == code if code == 2 else 4 <= got <= 13      # many rows: whichever of the block's warps gave up first
    assert pool.status() == 0
    check_attn(pool, q, seqs)
    assert pool.status() == 0


def test_attn_status_reports_both_kinds_of_block():
    lib = P().L.load()
    pool = random_pool(gen_of(57), 1, 10, 1, 64, 16, [100])
    q = torch.ones(20, 4, 64, device="cuda")
    lib.nsl_pages_attn_hold(1_000_000)
    try:
        pool.attn(0, q, ints([[0, 1, 99, 0]]), torch.empty_like(q), max_rows=1)
        pool.attn(0, q, ints([[0, 20, 80, 0]]), torch.empty_like(q), max_rows=20)
    finally:
        lib.nsl_pages_attn_hold(0)
    assert pool.status() == 2 and 4 <= pool.status() <= 13 and pool.status() == 0


# ---- warps that are partly filled ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,page", [(128, 64), (128, 16), (64, 32), (64, 128)])
@pytest.mark.parametrize("cols", [1, 3, 7, 8, 9, 15, 17, 31, 33, 47, 65, 96, 100, 127, 129, 130, 161, 200, 255, 257, 300])
def test_attn_of_any_number_of_columns(cols, hd, page):
    """Columns that end anywhere in a warp, some of which have their maxima move with every unit and others only with the first."""
    g = gen_of(cols + hd)
    n = max(500, cols + 200)
    pool = random_pool(g, 2, -(-n // page) + 1, 2, hd, page, [n])
    q = torch.randn(cols + 1, 2, hd, generator=g, device="cuda")
    k = held(pool, 1, 0, n)[0].float()      # [n][2][hd]
    grow = torch.arange(n, device="cuda")[:, None, None] / n
    pool.k[1, pool.table[0].long()] = 0
    pool.append(1, None, None, (k * grow ** 2).contiguous(), (torch.randn(n, 2, hd, generator=g, device="cuda")).contiguous(), ints([[0, n, 0, 0]]))
    q[::3] *= 0.01
    check_attn(pool, q.to(torch.bfloat16), [[0, cols, n - cols, 0]])


# ---- calls beside one another -----------------------------------------------------------------------------------------------------------
def calls_of(pool):
    """Two calls whose items are all dealt to several blocks, so that both keep states in their work memory."""
    g = gen_of(58)
    out = []
    for seqs in ([[0, 1, 2999, 0], [1, 1, 1999, 1]], [[0, 150, 2550, 0], [150, 3, 1900, 1]]):
        q = torch.randn(153, 16, 128, generator=g, device="cuda").to(torch.bfloat16)
        alone = torch.zeros_like(q)
        rows, most = ints(seqs), max(n for _, n, _, _ in seqs)
        pool.attn(1, q, rows, alone, max_rows=most)
        out.append((q, rows, most, alone))
    torch.cuda.synchronize()
    return out


def test_attn_on_two_streams_of_one_pool():
    pool = random_pool(gen_of(59), 2, 700, 2, 128, 16, [3000, 2000])
    calls = calls_of(pool)
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [[torch.zeros_like(q) for _ in range(10)] for q, _, _, _ in calls]
    torch.cuda.synchronize()
    for i in range(10):
        for (q, rows, most, _), stream, out in zip(calls, streams, outs):
            with torch.cuda.stream(stream):
                pool.attn(1, q, rows, out[i], max_rows=most)
    torch.cuda.synchronize()
    for (*_, alone), out in zip(calls, outs):
        assert all(torch.equal(o, alone) for o in out)
    handles = [s.cuda_stream for s in streams]
    works = [pool._works[h].data_ptr() for h in handles]
    assert len({*works, pool.attn_work.data_ptr()}) == 3
    with torch.cuda.stream(streams[0]):      # the stream's own from then on
        pool.attn(1, *calls[0][:2], outs[0][0], max_rows=calls[0][2])
    assert pool._works[handles[0]].data_ptr() == works[0]
    torch.cuda.synchronize()


def test_attn_in_two_graphs_replayed_beside_one_another():
    pool = random_pool(gen_of(59), 2, 700, 2, 128, 16, [3000, 2000])
    calls = calls_of(pool)
    graphs, outs, held_before = [], [], len(pool._works)
    for q, rows, most, _ in calls:
        out = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for layer in (0, 1, 0, 1):
                pool.attn(layer, q, rows, out, max_rows=most)
        graphs.append(graph)
        outs.append(out)
    assert len(pool._works) == held_before      # the memory is the graph's
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        pool.attn(1, calls[0][0], calls[0][1], torch.empty_like(outs[0]), max_rows=calls[0][2])      # and a call of the current stream's
        torch.cuda.synchronize()
        for out, (*_, alone) in zip(outs, calls):
            assert torch.equal(out, alone)


def test_host_tensors_are_refused():
    x, rows = torch.zeros(2, 2, 64), torch.zeros(1, 4, dtype=torch.int32)
    pool = P().PagePool.empty(1, 4, 2, 64, 16, 2, 2)
    y = x.cuda()
    for call in (lambda: P().rope(P().Rope(inv_of(64)), x, None, rows[0, :2]), lambda: P().rope(P().Rope(inv_of(64)), y, None, rows[0, :2]), lambda: pool.attn(0, x, rows.cuda(), x.clone(), max_rows=1),
                 lambda: pool.attn(0, y, rows.cuda(), torch.empty_like(y), max_rows=1, work=torch.zeros(1 << 24, dtype=torch.int32)), lambda: pool.trim(rows[:, :2].contiguous())):
        with pytest.raises(ValueError, match="the host|on cpu"):
            call()


# ---- outputs beside inputs ---------------------------------------------------------------------------------------------------------------
def test_outputs_in_place_and_beside_the_inputs():
    """Rows side by side in wider rows, behind one another, and in place are served; what overlaps is refused and nothing is written."""
    g = gen_of(60)
    pool = random_pool(g, 2, 30, 2, 64, 16, [100])
    wide = torch.randn(9, 4 * 512, generator=g, device="cuda").to(torch.bfloat16)
    cols = lambda i: wide[:, 512 * i:512 * i + 512].view(9, 8, 64)  # noqa: E731
    q, seqs = cols(1), [[0, 9, 60, 0]]
    want, size = attn64(pool, 1, q, seqs, 0.125, 0)
    for out in (cols(0), cols(2), cols(3)):
        pool.attn(1, q, ints(seqs), out, max_rows=9)
        assert bool(((out.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size).all())
    behind = torch.zeros(18, 8, 64, dtype=torch.bfloat16, device="cuda")
    behind[:9] = q
    pool.attn(1, behind[:9], ints(seqs), behind[9:], max_rows=9)
    assert torch.equal(behind[9:], cols(3)) and torch.equal(behind[:9], q)
    keep, r, pos = wide.clone(), P().Rope(inv_of(64)), ints(list(range(9)))
    k, v = torch.zeros(9, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(9, 2, 64, dtype=torch.bfloat16, device="cuda")
    flat = wide.flatten()
    part = lambda first: flat.as_strided((9, 8, 64), (2048, 64, 1), first)[:8]  # noqa: E731
    bad = [lambda: pool.attn(1, q, ints(seqs), q, max_rows=9), lambda: pool.attn(1, q[:8], ints(seqs), part(512 + 8), max_rows=9), lambda: pool.attn(1, q[:8], ints(seqs), q[1:], max_rows=9),
           lambda: P().rope(r, q[:8], None, pos[:8], part(512 + 64)), lambda: P().rope(r, q, cols(1)[:, :2], pos), lambda: P().rope(r, q, k, pos, cols(2), cols(2)[:, 4:6]),
           lambda: pool.append(1, r, q, k, cols(2)[:, :2], ints(seqs), cols(2)), lambda: pool.read(1, ints(seqs), cols(0)[:, :2], cols(0)[:, 1:3])]
    for call in bad:
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert torch.equal(wide, keep)
    P().rope(r, q, cols(2), pos, cols(1), cols(3))      # in place, and beside
    for a, b in ((1, 1), (2, 3)):
        x = keep[:, 512 * a:512 * a + 512].view(9, 8, 64)
        y, size = turned(x, pos, r.inv, False, 1.0)
        assert bool(((cols(b).double() - y).abs() <= 4 * F32 * size + BF16 * (y.abs() + 4 * F32 * size)).all())


# ---- whose refusal the handle raises -------------------------------------------------------------------------------------------------------
def test_a_served_call_raises_nothing():
    """Refusals that nobody has read, of this thread's other calls and of another thread's, are not the handle's."""
    lib, pool = P().L.load(), P().PagePool.empty(1, 8, 1, 64, 16, 2, 4)
    bad = lambda: lib.nsl_pages_fork(None, pool._p, None, 1)  # noqa: E731
    bad()
    t = threading.Thread(target=bad)
    t.start()
    t.join()
    x, rows = torch.randn(3, 1, 64, device="cuda"), ints([[0, 3, 0, 0]])
    pool.extend(ints([[0, 3]]))
    pool.append(0, None, None, x, x, rows)
    pool.attn(0, x, rows, torch.empty_like(x), max_rows=3)
    with pytest.raises(ValueError, match="nsl_pages_append"):
        pool.append(1, None, None, x, x, rows)
    assert P().L.last_error().startswith("nsl_pages_fork")


# ---- queries that are not finite ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,heads,hd,page", [(1, 8, 128, 64), (2, 8, 64, 16), (5, 8, 128, 16), (40, 8, 64, 64), (300, 4, 128, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_attn_of_queries_that_are_not_finite(rows, heads, hd, page, dtype, what):
    """The softmax of scores that hold a NaN, or an infinity times codes of both signs and 0, is NaN: so is that row's head, and nothing else; a row that
    nothing is left for gives zeros whatever its query holds."""
    g = gen_of(54)
    pool = random_pool(g, 2, 80, 2, hd, page, [900, 64])
    q = torch.randn(rows + 1, heads, hd, generator=g, device="cuda").to(torch.bfloat16).to(dtype)
    seqs = [[0, rows, 899 - rows, 0], [rows, 1, -4, 1]]
    a = check_attn(pool, q, seqs, out_dtype=dtype)
    bad = q.clone()
    bad[rows // 2, 1, 7] = what
    bad[rows, 0, 3] = what
    b = torch.full_like(a, 5.0)
    pool.attn(1, bad, ints(seqs), b, max_rows=rows)
    assert bool(b[rows // 2, 1].isnan().all()) and bool((b[rows] == 0).all())
    b[rows // 2, 1] = a[rows // 2, 1]
    assert torch.equal(a, b)


# ---- page scales far apart, masked pages and large pools, on both attention kernels and all page sizes ---------------------------------
FORMS = [(1, 4, 128, 64), (1, 4, 64, 16), (2, 4, 64, 128), (1, 8, 128, 16), (2, 2, 128, 128), (3, 8, 128, 64), (5, 8, 64, 128), (200, 4, 128, 128), (150, 2, 64, 64), (100, 8, 64, 32)]      # rows, heads a KV head, hd, page


@pytest.mark.parametrize("rows,group,hd,page", FORMS, ids=str)
def test_attn_scales_far_apart(rows, group, hd, page):
    g = gen_of(13 + rows + page)
    pool = random_pool(g, 2, 2 * (-(-700 // page)) + 3, 2, hd, page, [700, 300])
    pool.vs.copy_(torch.exp2(torch.randint(-60, 40, pool.vs.shape, generator=g, device="cuda").float()))
    pool.ks[:, ::5] = 0.0
    pool.vs[:, ::7] = 0.0
    q = torch.randn(2 * rows, 2 * group, hd, generator=g, device="cuda").to(torch.bfloat16)
    seqs = [[0, rows, 700 - rows, 0], [rows, rows, 250 - rows, 1]]
    check_attn(pool, q, seqs, scale=0.01)
    check_attn(pool, q, seqs, scale=0.01, window=page + 3)
    check_attn(pool, q * 0, seqs)
    pool.vs.copy_(torch.exp2(torch.arange(pool.vs.numel(), device="cuda").view(pool.vs.shape) % 120 - 110.0))      # up to 2^119 between neighbours
    check_attn(pool, q, seqs, scale=0.01)
    pool.vs.fill_(0.0)
    assert bool((check_attn(pool, q, seqs) == 0).all())


@pytest.mark.parametrize("rows,group,hd,page", FORMS, ids=str)
def test_attn_takes_nothing_from_masked_pages(rows, group, hd, page):
    """Scales and codes of pages outside the window or behind the last position may be anything."""
    g = gen_of(14 + rows + page)
    pool = random_pool(g, 2, 2 * (-(-1400 // page)) + 3, 2, hd, page, [1400, 1400])
    q = torch.randn(2 * rows, 2 * group, hd, generator=g, device="cuda").to(torch.bfloat16)
    at = 1000 // page * page - 1      # the last row's position is the last of its page
    seqs = [[0, rows, at - rows + 1, 0], [rows, rows, 700 - rows, 1]]
    a = check_attn(pool, q, seqs, window=100)
    dead = [pool.table[0, (at + 1) // page:], pool.table[1, 700 // page + 1:], pool.table[0, :(at - rows - 100) // page], pool.table[1, :max(0, 700 - rows - 100) // page]]
    for n, ids in enumerate(dead):
        for t in (pool.ks, pool.vs):
            t[:, ids.long()] = [float("nan"), float("inf"), -1.0, 0.0][n]
        pool.k[:, ids.long()] = 127
        pool.v[:, ids.long()] = -128
    b = check_attn(pool, q, seqs, window=100)
    assert torch.equal(a, b)
    # codes behind the last position, in its own page
    pool.k[:, pool.table[1, 700 // page].long(), :, 700 % page:] = 127
    pool.v[:, pool.table[1, 700 // page].long(), :, 700 % page:] = -127
    assert torch.equal(a, check_attn(pool, q, seqs, window=100))


@pytest.mark.parametrize("hd,page", [(128, 64), (128, 16), (64, 128)])
def test_attn_of_single_rows_beyond_32_bits(hd, page):
    """Pages more than 2^32 bytes into the pool, read by the kernel of few columns."""
    kv = 8
    pages = (1 << 32) // (kv * hd * page) + 2000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 20 GB")
    shape = (1, pages, kv, page, hd)
    k, v = (torch.empty(shape, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full(shape[:3], 2.0 ** -6, device="cuda") for _ in range(2))
    g = gen_of(16)
    ids = [pages - 1, 3, pages - 2, 7, pages - 1900]
    for i in ids:
        for t in (k, v):
            t[0, i] = torch.randint(-127, 128, shape[2:], generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    pool = P().PagePool(k, v, ks, vs, torch.ones(pages, dtype=torch.int32, device="cuda"), ints([ids, ids[::-1]]), ints([5 * page] * 2))
    q = torch.randn(2, 16, hd, generator=g, device="cuda").to(torch.bfloat16)
    check_attn(pool, q, [[0, 1, 5 * page - 1, 0], [1, 1, 3 * page + 2, 1]], layer=0)


# ---- queries with all of float32's bits ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,group,hd,page", [(1, 8, 128, 64), (1, 4, 64, 16), (2, 4, 64, 128), (1, 1, 128, 16), (6, 8, 64, 32), (3, 16, 128, 64), (70, 8, 128, 16), (200, 4, 128, 128), (150, 2, 64, 64)], ids=str)
@pytest.mark.parametrize("size", [1.0, 8.0, 32.0])
def test_attn_float32_queries(rows, group, hd, page, size):
    """Queries with 24 significant bits: the tolerance has no term for them.  Scores are as large as the queries make them, so their f32 sums' share grows with
    size: hd products, each rounded once more in the sum (2^-24 of sum |q k| scale each), and 2^-24 of the largest query by the keys' sum for the queries themselves."""
    g = gen_of(rows + page + int(size))
    n = 1500
    pool = random_pool(g, 2, -(-n // page) + 2, 2, hd, page, [n])
    pool.ks.fill_(2.0 ** -6)
    pool.k.copy_((torch.randn(pool.k.shape, generator=g, device="cuda") * 36).round().clamp(-127, 127).to(torch.int8))
    q = torch.randn(rows, 2 * group, hd, generator=g, device="cuda") * size
    seqs = [[0, rows, n - rows, 0]]
    o = torch.full(q.shape, 5.0, device="cuda")
    pool.attn(1, q, ints(seqs), o, max_rows=rows)
    want, total = attn64(pool, 1, q, seqs, hd ** -0.5, 0)
    scale = hd ** -0.5
    k = held(pool, 1, 0, n)[0]      # [n][kv][hd]
    s = torch.einsum("ngd,rgjd->rgjn", k.abs(), q.double().abs().view(rows, 2, group, hd)).amax(-1) * scale      # the largest sum |q k| scale of a column
    top = (q.double().abs().amax(-1).view(rows, 2, group) * k.abs().sum(-1).amax(0)[None, :, None]) * scale
    off = 2 * (hd * F32 * s + 2 * F32 * top + 4 * F32 * s)      # of a weight, relative: in numerator and sum
    # a weight times its page's value scale is held as f16: 2^-11 of it, or, below 2^-14 of the largest such product, half a subnormal step, 2^-25 of the
    # largest, by the code that it multiplies.  That is next to nothing of the row, but can be all of an element to which the heaviest keys add codes of 0.
    p64 = torch.einsum("ngd,rgjd->rgjn", k, q.double().view(rows, 2, group, hd)) * scale
    p64 = p64.masked_fill(torch.arange(n, device="cuda") > torch.arange(n - rows, n, device="cuda")[:, None, None, None], -math.inf).softmax(-1)
    at = torch.arange(n, device="cuda")
    vs = pool.vs[1, pool.table[0, at // page].long()].double()      # [n][kv]
    most = (p64 * vs.T[None, :, None]).amax(-1)      # [rows][kv][group]
    codes = (held(pool, 1, 0, n)[1] / vs[..., None]).abs().sum(0)      # [kv][hd]
    small = 2.0 ** -25 * (most[..., None] * codes[None, :, None]).reshape(rows, 2 * group, hd)
    tol = ((2.0 ** -11 + off.view(rows, 2 * group, 1)) * total + small) * (1 + BF16) + BF16 * want.abs()
    far = ((o.double() - want).abs() / tol).max()
    assert float(far) <= 1.0


@pytest.mark.parametrize("rows,group,hd,page", [(1, 8, 128, 64), (6, 8, 64, 32), (200, 4, 128, 16)], ids=str)
def test_attn_float32_arrays_of_bf16_values(rows, group, hd, page):
    """The same bits as bf16 queries, said to be rounded or not."""
    g = gen_of(61)
    pool = random_pool(g, 2, -(-900 // page) + 2, 2, hd, page, [900])
    q = torch.randn(rows, 2 * group, hd, generator=g, device="cuda").to(torch.bfloat16)
    rows_, outs = ints([[0, rows, 900 - rows, 0]]), []
    for x, more in ((q, {}), (q.float(), {}), (q.float(), {"rounded": True})):
        outs.append(torch.empty_like(q))
        pool.attn(1, x, rows_, outs[-1], max_rows=rows, **more)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- calls that the documentation allows and the other tests do not make -----------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,rows", [(300, 1, 1), (272, 1, 3), (1040, 2, 1), (600, 2, 2)])
def test_attn_of_more_heads_than_an_item_has_columns(heads, kv, rows):
    g = gen_of(heads)
    pool = random_pool(g, 2, 30, kv, 64, 32, [500, 90])
    q = torch.randn(2 * rows, heads, 64, generator=g, device="cuda").to(torch.bfloat16)
    check_attn(pool, q, [[0, rows, 500 - rows, 0], [rows, rows, 90 - rows, 1]])
    check_attn(pool, q, [[0, rows, 500 - rows, 0], [rows, rows, 90 - rows, 1]], window=70)


@pytest.mark.parametrize("n,heads", [(1000, 16), (4096, 16), (4096, 4)])
def test_attn_padded_batches_of_many_sequences(n, heads):
    """Every third place of the batch is empty, in either attention kernel; the list is as long as it may be."""
    g = gen_of(n)
    lens = [1 + (53 * i) % 200 for i in range(n)]
    pool = random_pool(g, 2, sum(-(-m // 32) for m in lens), 1, 64, 32, lens)
    q = torch.randn(n, heads, 64, generator=g, device="cuda").to(torch.bfloat16)
    check_attn(pool, q, [[i, 0 if i % 3 == 1 else 1, m - 1, i] for i, m in enumerate(lens)])


def test_append_of_many_rows_with_heads_that_do_not_divide():
    """Blocks with several rows of queries and several of the three KV heads; read back with several rows a block."""
    g = gen_of(62)
    kv, hd, page, seqs = 3, 64, 16, [(5, 9000), (0, 1), (31, 500), (16, 16)]
    lengths = [p + n for p, n in seqs]
    pool = random_pool(g, 2, sum(-(-m // page) for m in lengths) + 3, kv, hd, page, lengths)
    T = sum(n for _, n in seqs)
    q, k, v = (torch.randn(T, h, hd, generator=g, device="cuda").to(torch.bfloat16) for h in (5, kv, kv))
    desc, row = [], 0
    for s, (p, n) in enumerate(seqs):
        desc += [[row, n, p, s], [T, 5, 3, 1]]      # and places behind the call's rows
        row += n
    before = [(a.clone(), b.clone()) for a, b in ((pool.k, pool.ks), (pool.v, pool.vs))]
    r, qo = P().Rope(inv_of(32)), torch.empty_like(q)
    pool.append(1, r, q, k, v, ints(desc), qo)
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in seqs])
    for x, got in ((q, qo),):
        want, size = turned(x, pos, r.inv, False, 1.0)
        assert bool(((got.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * 4 * F32 * size).all())
    kr, size = turned(k, pos, r.inv, False, 1.0)
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    pool.read(1, ints(desc), kb, vb)
    for codes, scales, was, x, tol, back in ((pool.k, pool.ks, before[0], kr, 4 * F32 * size, kb), (pool.v, pool.vs, before[1], v.double(), 0 * size, vb)):
        row = 0
        for s, (p, n) in enumerate(seqs):
            ids, at = pool.table[s].long(), torch.arange(p, p + n, device="cuda")
            pid = ids[at // page]
            scale = scales[1, pid].double()      # [n][kv]
            mine = x[row:row + n]
            # of each page: the power of two for its new rows, or the old scale where rows were there before and theirs was larger
            top = torch.zeros(codes.shape[1], kv, dtype=torch.float64, device="cuda").scatter_reduce(0, pid[:, None].expand(-1, kv), mine.abs().amax(-1), "amax")
            m, e = torch.frexp(top)      # top = m 2^e, m in [1/2, 1): top <= 127 2^(e - 7) where m <= 127 / 128
            need = torch.ldexp(torch.ones_like(top), torch.where(m <= 127 / 128, e - 7, e - 6))
            first = int(ids[p // page])
            if p % page:
                need[first] = torch.maximum(need[first], was[1][1, first].double())
            assert torch.equal(scale, need[pid])
            held_now = codes[1, pid, :, at % page].double() * scale[..., None]
            assert bool(((held_now - mine).abs() <= scale[..., None] / 2 + tol[row:row + n]).all())
            assert torch.equal(back[row:row + n], held_now.float().to(torch.bfloat16))
            row += n


def test_a_captured_step_is_replayed_with_other_lengths():
    """Management, store and attention captured into one graph, and replayed with descriptors and requests that are changed on the device, against the same
    calls one by one on another pool."""
    g = gen_of(63)
    def build():
        pool = P().PagePool.empty(2, 60, 2, 64, 16, 4, 12)
        for t in (pool.k, pool.v, pool.ks, pool.vs):
            t.zero_()
        return pool
    a, b = build(), build()
    x = torch.randn(12, 3, 4, 8, 64, generator=g, device="cuda").to(torch.bfloat16)
    r = P().Rope(inv_of(64))
    ins = [x[0, i].clone() for i in range(3)]
    rows, grow, forks, cut = ints([[0, 1, 0, 0], [1, 3, 0, 1], [0, 0, 0, 2], [0, 0, 0, 3]]), ints([[0, 1], [1, 3]]), ints([[0, 2, 0, 0]]), ints([[3, 0]])
    qa, oa = torch.zeros(4, 8, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 8, 64, dtype=torch.bfloat16, device="cuda")

    def step(pool, q2, o):
        pool.trim(cut)
        pool.fork(forks)
        pool.extend(grow)
        for layer in (0, 1):
            pool.append(layer, r, ins[0], ins[1][:, :2], ins[2][:, :2], rows, q2)
            pool.attn(layer, q2, rows, o, max_rows=3)
        pool.compact()

    graph = torch.cuda.CUDAGraph()
    state = [t.clone() for t in (a.table, a.ref, a.length)]
    with torch.cuda.graph(graph):
        step(a, qa, oa)
    for t, was in zip((a.table, a.ref, a.length), state):
        assert torch.equal(t, was)      # capturing runs nothing
    length = {0: 0, 1: 0}
    for i in range(12):
        for j in range(3):
            ins[j].copy_(x[i, j])
        plan = [[0, 1, length[0], 0], [1, 3, length[1], 1], [0, 0, 0, 2], [0, 0, 0, 3]]
        rows.copy_(ints(plan))
        length[0], length[1] = length[0] + 1, length[1] + 3
        grow.copy_(ints([[0, length[0]], [1, length[1]]]))
        forks.copy_(ints([[1, 2, 9, 0] if i == 5 else [0, 0, 0, 0]]))
        cut.copy_(ints([[2, 0] if i == 9 else [1, length[1]]]))
        graph.replay()
        qb, ob = torch.zeros_like(qa), torch.zeros_like(oa)
        step(b, qb, ob)
        assert torch.equal(oa, ob) and torch.equal(qa, qb)
        for s, t in ((a.table, b.table), (a.ref, b.ref), (a.length, b.length)):
            assert torch.equal(s, t)
        want, size = attn64(a, 1, qa, plan, 0.125, 0)
        assert bool(((oa.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size).all())


@pytest.mark.parametrize("offset", [0, 1, 37])
def test_lists_anywhere_in_memory(offset):
    """Descriptors and requests of odd offsets in a longer list: 4-byte alignment is all they have."""
    g = gen_of(64)
    pool = random_pool(g, 2, 20, 2, 64, 16, [100, 60])
    q = torch.randn(6, 8, 64, generator=g, device="cuda").to(torch.bfloat16)
    seqs = [[0, 1, 99, 0], [1, 5, 40, 1]]
    flat = torch.zeros(offset + 8, dtype=torch.int32, device="cuda")
    flat[offset:] = ints(seqs).flatten()
    check_attn(pool, q, seqs, rows=flat[offset:].view(2, 4))
