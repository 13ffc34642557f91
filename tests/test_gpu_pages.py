"""The paged 8-bit cache on the GPU against plain implementations in 64 bits: rotary positions, the store and the read back,
attention over pages, the pages' management, and a run of them together.

Roundings that the tolerances count (half a step each, relative): f32 2^-24, bf16 2^-8, f16 2^-11."""
import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = 2.0 ** -24, 2.0 ** -8


def P():
    from nanoseedlm_b200 import pages
    return pages


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inv_of(rot, theta=1e6):
    return torch.tensor([theta ** (-2.0 * p / rot) for p in range(rot // 2)], dtype=torch.float64).float().cuda()


# ---- rotary positions ---------------------------------------------------------------------------------------------------------
def turned(x, pos, inv, inter, factor):
    """x [T][heads][hd] rotated, in 64 bits; and |u| + |w| of each value's pair, 0 where nothing is rotated."""
    x = x.double()
    rot, a = 2 * inv.numel(), pos.double()[:, None] * inv.double()
    cs, sn = (factor * a.cos())[:, None], (factor * a.sin())[:, None]
    y, size = x.clone(), torch.zeros_like(x)
    at = torch.arange(inv.numel(), device="cuda")
    i, j = (2 * at, 2 * at + 1) if inter else (at, at + rot // 2)
    u, w = x[..., i], x[..., j]
    y[..., i], y[..., j] = u * cs - w * sn, w * cs + u * sn
    size[..., i] = size[..., j] = u.abs() + w.abs()
    return y, size


# An angle reduced to half a turn is below 4, its rounding to f32 off by 2^-23 at most; sine and cosine by 2 units more (4 F32), their
# product with the factor, the two products and the sum by 4 F32: 10 F32 of factor (|u| + |w|).
ROPE = 10 * F32


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,heads,kv,hd,rot,typ", [(1, 1, 0, 16, 16, "f32"), (1, 16, 2, 128, 128, "bf16"), (3, 5, 1, 64, 32, "f32"), (7, 16, 2, 128, 64, "rounded"), (33, 2, 2, 256, 64, "bf16"),
                                                   (130, 3, 1, 512, 512, "f32"), (2500, 8, 4, 64, 48, "bf16")])
def test_rope(T, heads, kv, hd, rot, typ, inter):
    g = gen_of(T + rot)
    dt = torch.float32 if typ == "f32" else torch.bfloat16
    mk = lambda n: (torch.randn(T, n, hd, generator=g, device="cuda") * 3).to(dt).to(torch.float32 if typ != "bf16" else dt)  # noqa: E731
    q, k = mk(heads), mk(kv) if kv else None
    pos = torch.randint(-5, 2 ** 31 - 1, (T,), generator=g, device="cuda", dtype=torch.int32)      # every int32 position
    inv, factor = inv_of(rot), 1.3
    r = P().Rope(inv, interleaved=inter, factor=factor)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0) if kv else None
    P().rope(r, q, k, pos, qo, ko, rounded=typ == "rounded")
    q2, k2 = q.clone(), k.clone() if kv else None
    P().rope(r, q2, k2, pos, rounded=typ == "rounded")      # in place
    for x, got, again in ((q, qo, q2), (k, ko, k2)):
        if x is None:
            continue
        want, size = turned(x, pos, inv, inter, factor)
        tol = ROPE * factor * size + (0 if typ == "f32" else BF16 * (want.abs() + ROPE * factor * size))
        assert bool(((got.double() - want).abs() <= tol).all())
        assert torch.equal(got, again)
        assert torch.equal(got[..., rot:], x[..., rot:])
        if typ == "rounded":
            assert torch.equal(got, got.to(torch.bfloat16).float())


def test_rope_strides_and_rows_left_alone():
    g = gen_of(5)
    big = torch.randn(9, 3 * 8 * 64, generator=g, device="cuda").to(torch.bfloat16)      # q, k, v side by side in a row
    keep = big.clone()
    q, k = big[:, :512].view(9, 8, 64), big[:, 512:1024].view(9, 8, 64)
    inv, pos = inv_of(64), ints(list(range(9)))
    P().rope(P().Rope(inv), q[:6], k[:6], pos[:6])
    for a, b in ((0, 512), (512, 1024)):
        want, size = turned(keep[:6, a:b].reshape(6, 8, 64), pos[:6], inv, False, 1.0)
        assert bool(((big[:6, a:b].reshape(6, 8, 64).double() - want).abs() <= ROPE * size + BF16 * (want.abs() + ROPE * size)).all())
    assert torch.equal(big[6:], keep[6:]) and torch.equal(big[:, 1024:], keep[:, 1024:])


def test_rope_takes_non_finite_values_along():
    x = torch.zeros(1, 2, 64, device="cuda")
    x[0, 0, 3], x[0, 1, 5] = float("nan"), float("inf")
    P().rope(P().Rope(inv_of(64)), x, None, ints([9]))
    bad = ~torch.isfinite(x)
    assert bad[0, 0].nonzero().flatten().tolist() == [3, 35] and bad[0, 1].nonzero().flatten().tolist() == [5, 37]


# ---- pools --------------------------------------------------------------------------------------------------------------------
def random_pool(g, layers, n_pages, kv, hd, page, lengths, max_pages=None, pow2=True):
    """A pool with sequences of the given lengths (pages in a random order), codes and scales random."""
    shape = (layers, n_pages, kv, page, hd)
    codes = lambda: torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)  # noqa: E731
    if pow2:
        scales = lambda: torch.exp2(torch.randint(-8, -4, shape[:3], generator=g, device="cuda").float())  # noqa: E731
    else:
        scales = lambda: torch.rand(shape[:3], generator=g, device="cuda") * 0.03 + 0.001  # noqa: E731
    need = [-(-n // page) for n in lengths]
    max_pages = max_pages or max(need + [1])
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    table, ref, at = torch.full((len(lengths), max_pages), -1, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        ref[ids[at:at + n].long()] = 1
        at += n
    return P().PagePool(codes(), codes(), scales(), scales(), ref, table, ints(lengths))


def held(pool, layer, seq, n):
    """Keys and values of a sequence's first n positions in 64 bits: [n][kv][hd]."""
    ids = pool.table[seq, :-(-n // pool.page)].long()
    out = []
    for codes, scales in ((pool.k, pool.ks), (pool.v, pool.vs)):
        x = codes[layer, ids].double() * scales[layer, ids].double()[..., None, None]
        out.append(x.permute(0, 2, 1, 3).reshape(-1, pool.kv, pool.hd)[:n])
    return out


# ---- the store ----------------------------------------------------------------------------------------------------------------
def scale_for(top):
    """The smallest power of two (from 2^-126) with top <= 127 scale."""
    e = -126
    while top > 127 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def check_store(pool, before, layer, pos, rows_of, x_of, tol_of, which):
    """What pages hold after a call: pages' scales as defined, new rows within half a step of x, old ones within half a step of what they
    were, everything else untouched."""
    codes, scales = (pool.k, pool.ks) if which == "k" else (pool.v, pool.vs)
    codes0, scales0 = before
    touched = torch.zeros(codes.shape[1], dtype=torch.bool, device="cuda")
    for seq, (p0, n) in rows_of.items():
        for j in range(p0 // pool.page, (p0 + n - 1) // pool.page + 1):
            pid = int(pool.table[seq, j])
            touched[pid] = True
            lo, hi = max(p0, j * pool.page), min(p0 + n, (j + 1) * pool.page)
            x, tol = x_of[seq][lo - p0:hi - p0], tol_of[seq][lo - p0:hi - p0]
            off = lo - j * pool.page
            for h in range(pool.kv):
                need = scale_for(float(x[:, h].abs().max()))
                old = float(scales0[layer, pid, h]) if off else 0.0
                s = max(need, old)
                assert float(scales[layer, pid, h]) == s, (seq, j, h)
                new = codes[layer, pid, h, off:off + hi - lo].double() * s
                assert bool(((new - x[:, h]).abs() <= s / 2 + tol[:, h] + 1e-30).all())
                was = codes0[layer, pid, h, :off].double() * old
                now = codes[layer, pid, h, :off].double() * s
                assert bool(((now - was).abs() <= (s / 2 if s > old else 0)).all())
                if s == old:
                    assert torch.equal(codes[layer, pid, h, :off], codes0[layer, pid, h, :off])
                assert torch.equal(codes[layer, pid, h, off + hi - lo:], codes0[layer, pid, h, off + hi - lo:])
    rest = ~touched
    assert torch.equal(codes[:, rest], codes0[:, rest]) and torch.equal(scales[:, rest], scales0[:, rest])
    others = [l for l in range(codes.shape[0]) if l != layer]
    assert torch.equal(codes[others], codes0[others]) and torch.equal(scales[others], scales0[others])


STORES = [  # kv, hd, page, rot, interleaved, type, [(position, rows)] by sequence
    (2, 128, 64, 128, False, "f32", [(0, 1)]),
    (2, 128, 64, 128, False, "f32", [(63, 1), (64, 1), (17, 1), (0, 1), (128, 1)]),
    (1, 64, 16, 16, True, "bf16", [(5, 40), (0, 16), (31, 1), (15, 2)]),
    (4, 64, 32, 64, False, "bf16", [(0, 333), (100, 77)]),
    (3, 128, 128, 64, True, "rounded", [(120, 300), (0, 129)]),
    (8, 128, 128, 128, False, "f32", [(3, 1), (127, 5), (255, 130)]),
    (2, 64, 64, 0, False, "bf16", [(10, 70)]),
]


@pytest.mark.parametrize("kv,hd,page,rot,inter,typ,seqs", STORES, ids=str)
def test_append_and_read(kv, hd, page, rot, inter, typ, seqs):
    g = gen_of(kv * hd + page)
    lengths = [p + n for p, n in seqs]
    pool = random_pool(g, 2, sum(-(-n // page) for n in lengths) + 3, kv, hd, page, lengths)
    T, heads = sum(n for _, n in seqs), 2 * kv
    dt = torch.bfloat16 if typ == "bf16" else torch.float32
    size = torch.rand(T, 1, 1, generator=g, device="cuda") * 6      # rows of very different sizes: scales grow within a page
    mk = lambda n: (torch.randn(T, n, hd, generator=g, device="cuda") * torch.exp2(size)).to(dt)  # noqa: E731
    q, k, v = mk(heads), mk(kv), mk(kv)
    inv = inv_of(rot) if rot else None
    r = P().Rope(inv, interleaved=inter) if rot else None
    order = list(range(len(seqs)))
    random.Random(3).shuffle(order)      # descriptors in any order, an empty place among them
    desc, row, at = [[0, 0, 0, 0]] * len(seqs), 0, {}
    for i, (p, n) in enumerate(seqs):
        desc[order[i]], at[i] = [row, n, p, i], row
        row += n
    desc = ints(desc[:1] + [[0, 0, 0, 0]] + desc[1:] + [[5, -3, 2, 1]])
    before_k, before_v = (pool.k.clone(), pool.ks.clone()), (pool.v.clone(), pool.vs.clone())
    qo = torch.full_like(q, 7.0)
    pool.append(1, r, q, k, v, desc, qo, rounded=typ == "rounded")
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in seqs])
    none = torch.zeros_like(k, dtype=torch.float64)
    kr, ksize = turned(k, pos, inv, inter, 1.0) if rot else (k.double(), none)
    qr, qsize = turned(q, pos, inv, inter, 1.0) if rot else (q.double(), torch.zeros_like(q, dtype=torch.float64))
    tol = ROPE * qsize + (0 if typ == "f32" else BF16 * (qr.abs() + ROPE * qsize))
    assert bool(((qo.double() - qr).abs() <= tol).all())
    rows_of = {i: s for i, s in enumerate(seqs)}
    cut = lambda x: {i: x[at[i]:at[i] + n] for i, (_, n) in enumerate(seqs)}  # noqa: E731
    check_store(pool, before_k, 1, pos, rows_of, cut(kr), cut(ROPE * ksize), "k")
    check_store(pool, before_v, 1, pos, rows_of, cut(v.double()), cut(none), "v")
    # read back: the codes times the scales, unrounded or rounded once; rows that no descriptor names stay
    kb, vb = (torch.full((T + 3, kv, hd), 9.0, dtype=dt, device="cuda") for _ in range(2))
    pool.read(1, desc, kb, vb, rounded=typ == "rounded")
    for i, (p, n) in enumerate(seqs):
        for got, want in zip((kb, vb), held(pool, 1, i, p + n)):
            want = want[p:].float()
            want = want if typ == "f32" else want.to(torch.bfloat16).to(dt)
            assert torch.equal(got[at[i]:at[i] + n], want)
    assert bool((kb[T:] == 9.0).all()) and bool((vb[T:] == 9.0).all())


def test_append_row_by_row_ends_with_the_scales_of_one_call():
    g = gen_of(77)
    x = torch.randn(100, 2, 64, generator=g, device="cuda") * torch.exp2(torch.rand(100, 1, 1, generator=g, device="cuda") * 8 - 4)
    a, b = (random_pool(gen_of(1), 1, 8, 2, 64, 32, [100]) for _ in range(2))
    a.append(0, None, None, x, -x, ints([[0, 100, 0, 0]]))
    for t in range(100):
        b.append(0, None, None, x[t:t + 1], -x[t:t + 1], ints([[0, 1, t, 0]]))
    used = a.table[0, :4].long()
    assert torch.equal(a.ks[:, used], b.ks[:, used]) and torch.equal(a.vs[:, used], b.vs[:, used])
    for p, q in zip(held(a, 0, 0, 100), held(b, 0, 0, 100)):
        # a value is rounded once to its page's last scale, and before to smaller ones, each half the next at most: less than one step in all
        step = a.ks[0, used].double()[torch.arange(100, device="cuda") // 32][..., None]
        assert bool(((p - q).abs() <= 1.5 * step).all())


def test_append_non_finite_and_extreme_values():
    pool = random_pool(gen_of(2), 1, 4, 2, 64, 16, [16])
    x = torch.zeros(3, 2, 64, device="cuda")
    x[0, 0, :4] = torch.tensor([float("nan"), 1.0, -3.0, 0.5])
    x[1, 1, :3] = torch.tensor([float("inf"), -float("inf"), 1e38])
    v = torch.full((3, 2, 64), 1e-45, device="cuda")      # the smallest subnormal: stored as 0 with the smallest scale
    v[:, 1] = 3.4e38
    pool.append(0, None, None, x, v, ints([[0, 3, 0, 0]]))
    pid = int(pool.table[0, 0])
    assert float(pool.ks[0, pid, 0]) == 2.0 ** -5 and pool.k[0, pid, 0, 0, :4].tolist() == [0, 32, -96, 16]
    assert float(pool.ks[0, pid, 1]) == 2.0 ** 122 and pool.k[0, pid, 1, 1, :2].tolist() == [127, -127]
    assert float(pool.vs[0, pid, 0]) == 2.0 ** -126 and bool((pool.v[0, pid, 0, :3] == 0).all())
    assert float(pool.vs[0, pid, 1]) == 2.0 ** 122 and bool((pool.v[0, pid, 1, :3].float() * 2.0 ** 122 > 3.3e38).all())


def test_append_to_absent_pages_stores_nothing():
    pool = random_pool(gen_of(3), 1, 6, 1, 64, 16, [40, 20], max_pages=3)
    pool.table[0, 1] = -1
    pool.table[1, 0] = 6      # one beyond the pool
    keep = [t.clone() for t in (pool.k, pool.v, pool.ks, pool.vs)]
    x = torch.randn(200, 1, 64, device="cuda")
    q = torch.ones(200, 1, 64, device="cuda")
    bad = ints([[0, 16, 16, 0], [16, 4, 0, 1], [20, 60, 48, 0], [80, 3, -2, 0], [100, 5, 0, 2], [110, 5, 0, -1], [190, 100, 32, 1], [-7, 9, 2147483000, 0]])
    pool.append(0, None, None, x, x, bad)
    # what has a page is stored: sequence 0's position 0 (the last of rows -2 .. 0)
    pid = int(pool.table[0, 0])
    assert torch.equal(pool.k[0, pid, 0, 1:], keep[0][0, pid, 0, 1:]) and not torch.equal(pool.k[0, pid, 0, 0], keep[0][0, pid, 0, 0])
    others = [i for i in range(6) if i != pid]
    for t, was in zip((pool.k, pool.v, pool.ks, pool.vs), keep):
        assert torch.equal(t[:, others], was[:, others])
    kb, vb = torch.full_like(x, 9.0), torch.full_like(x, 9.0)
    pool.read(0, bad, kb, vb)
    named = (kb != 9.0).any(-1).flatten().nonzero().flatten().tolist()
    assert named == [82]
    assert bool((q == 1).all())


# ---- attention ----------------------------------------------------------------------------------------------------------------
def attn64(pool, layer, q, seqs, scale, window):
    """-> o in 64 bits and sum p |v|, both [T][heads][hd]; seqs: [(first row, rows, position, sequence)]."""
    o, size = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    group = q.shape[1] // pool.kv
    for row, n, p, s in seqs:
        if n <= 0 or p + n <= 0:
            continue
        ids = pool.table[s].long()
        there = (ids >= 0) & (ids < pool.k.shape[1])
        at = torch.where(there, ids, 0)
        k, v = (codes[layer, at].double() * scales[layer, at].double()[..., None, None] for codes, scales in ((pool.k, pool.ks), (pool.v, pool.vs)))
        k, v = (x.permute(1, 0, 2, 3).reshape(pool.kv, -1, pool.hd) for x in (k, v))
        key, pos = torch.arange(k.shape[1], device="cuda"), torch.arange(p, p + n, device="cuda")
        seen = (key <= pos[:, None]) & there.repeat_interleave(pool.page)
        if window > 0:
            seen &= key > pos[:, None] - window
        x = q[row:row + n].double().view(n, pool.kv, group, pool.hd)
        w = torch.einsum("nghd,gkd->nghk", x, torch.nan_to_num(k)) * scale
        w = w.masked_fill(~seen[:, None, None], -math.inf).softmax(-1).nan_to_num(0.0)      # a row that sees nothing: zeros
        v = torch.nan_to_num(v)
        o[row:row + n] = torch.einsum("nghk,gkd->nghd", w, v).reshape(n, -1, pool.hd)
        size[row:row + n] = torch.einsum("nghk,gkd->nghd", w, v.abs()).reshape(n, -1, pool.hd)
    return o, size


# Weights are rounded to 11 bits (2^-11) and their sums taken unrounded; scores are f32 sums of hd products, off by at most
# hd 2^-24 sum |q k| scale, which is below 2^-12 for the inputs here (sum |q k| scale below 16 on average), and enter weights as
# exponents, in numerator and sum: 2 * 2^-12.  Together 2^-10 of sum p |v|; then the result's rounding to bf16.
WEIGHTS = 2.0 ** -10


def check_attn(pool, q, seqs, window=0, scale=None, layer=1, out_dtype=torch.bfloat16, max_rows=None, rows=None):
    T = q.shape[0]
    o = torch.full(q.shape, 5.0, dtype=out_dtype, device="cuda")
    scale = pool.hd ** -0.5 if scale is None else scale
    pool.attn(layer, q, ints(seqs) if rows is None else rows, o, max_rows=max_rows or max(n for _, n, _, _ in seqs), scale=scale, window=window)
    want, size = attn64(pool, layer, q, seqs, scale, window)
    named = torch.zeros(T, dtype=torch.bool, device="cuda")
    for row, n, _, _ in seqs:
        named[row:row + max(n, 0)] = True
    far = ((o.double() - want).abs() - BF16 * want.abs() - (1 + BF16) * WEIGHTS * size)[named]
    assert far.numel() == 0 or float(far.max()) <= 1e-30, float(far.max())
    assert bool((o[~named] == 5.0).all())
    if out_dtype == torch.float32:
        assert torch.equal(o, o.to(torch.bfloat16).float())
    return o


def some_rows(seqs):
    out, row = [], 0
    for s, (p, n) in enumerate(seqs):
        out.append([row, n, p, s])
        row += n
    return out, row


ATTN = [  # heads, kv, hd, page, window, [(position of the first row, rows)]
    (16, 2, 128, 64, 0, [(0, 1)]),
    (16, 2, 128, 64, 0, [(899, 1)]),
    (16, 2, 128, 64, 0, [(63, 1), (64, 1), (127, 1), (1, 1), (1000, 1), (0, 1), (513, 1)]),
    (8, 8, 64, 16, 0, [(700, 1), (15, 1), (16, 1)]),
    (16, 1, 128, 32, 0, [(333, 1), (2049, 1)]),
    (40, 8, 128, 128, 0, [(4095, 1), (4096, 1)]),
    (12, 4, 64, 32, 0, [(5, 3), (100, 6), (0, 1), (30, 2)]),
    (32, 4, 64, 32, 0, [(2000, 4), (31, 8), (0, 8)]),
    (32, 1, 128, 64, 0, [(600, 1), (70, 3)]),
    (64, 1, 64, 16, 0, [(100, 5)]),
    (16, 2, 128, 64, 0, [(0, 300)]),
    (16, 2, 128, 64, 0, [(777, 129), (5000, 1), (0, 17), (64, 64)]),
    (6, 3, 64, 128, 0, [(127, 130), (3, 1)]),
    (8, 8, 128, 16, 0, [(33, 200)]),
    (16, 2, 128, 64, 100, [(899, 1), (50, 1), (99, 1), (100, 1)]),
    (16, 2, 128, 64, 1, [(70, 3), (0, 1)]),
    (8, 2, 64, 16, 37, [(0, 150), (400, 40)]),
    (16, 2, 128, 64, 500, [(1200, 300)]),
]


@pytest.mark.parametrize("heads,kv,hd,page,window,seqs", ATTN, ids=str)
@pytest.mark.parametrize("typ", ["bf16", "f32"])
def test_attn(heads, kv, hd, page, window, seqs, typ):
    g = gen_of(heads + hd + page)
    lengths = [p + n for p, n in seqs]
    pool = random_pool(g, 2, sum(-(-n // page) for n in lengths) + 2, kv, hd, page, lengths, pow2=typ == "bf16")
    rows, T = some_rows(seqs)
    q = torch.randn(T + 2, heads, hd, generator=g, device="cuda").to(torch.bfloat16)
    q = q if typ == "bf16" else q.float()
    check_attn(pool, q, rows, window, out_dtype=q.dtype)


def test_attn_rows_that_see_nothing():
    g = gen_of(11)
    pool = random_pool(g, 2, 20, 2, 128, 16, [100, 50, 33], max_pages=8)
    pool.table[1] = -1                    # a sequence without pages
    pool.table[0, 1:] = 99                # ids beyond the pool
    pool.table[2, 1] = -1                 # a hole
    q = torch.randn(40, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    seqs = [[0, 5, 45, 1], [5, 3, 97, 0], [8, 4, 29, 2], [20, 0, 3, 0], [12, 2, -5, 0], [30, 2, 1000, 2]]
    o = check_attn(pool, q, seqs[:3] + [seqs[3], [14, 3, -2, 0]])
    assert bool((o[:5] == 0).all())
    assert bool((o[14:16] == 0).all()) and bool((o[16] != 0).any())      # positions -2 and -1; position 0
    o = check_attn(pool, q, seqs[:5], window=4)
    assert bool((o[5:8] == 0).all()) and bool((o[12:14] == 0).all())
    # positions beyond the table's row are left out like any without a page
    o = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device="cuda")
    pool.attn(1, q, ints([[30, 2, 1000, 2], [0, 2, 10, 3], [2, 2, 10, -1]]), o, max_rows=2)
    want, size = attn64(pool, 1, q, [[30, 2, 1000, 2]], 128 ** -0.5, 0)
    assert bool(((o.double() - want).abs()[30:32] <= (BF16 * want.abs() + (1 + BF16) * WEIGHTS * size)[30:32]).all())
    assert bool((o[:4] == 0).all()) and bool((o[4:30] == 5.0).all())


def test_attn_ignores_what_is_masked():
    """Scales of pages that no position of the row lies in may be anything, and so may codes behind the last position."""
    g = gen_of(12)
    pool = random_pool(g, 2, 30, 2, 64, 16, [64, 200])
    q = torch.randn(6, 8, 64, generator=g, device="cuda").to(torch.bfloat16)
    seqs = [[0, 1, 20, 0], [1, 5, 150, 1]]
    a = check_attn(pool, q, seqs, window=60)
    for scales in (pool.ks, pool.vs):
        scales[:, pool.table[0, 2:4].long()] = float("nan")
        scales[:, pool.table[1, :5].long()] = float("inf")      # positions 0 .. 79: the window of 150 begins at 91
    pool.k[:, pool.table[0, 1].long(), :, 5:] = 127
    pool.v[:, pool.table[0, 1].long(), :, 5:] = -127
    b = check_attn(pool, q, seqs, window=60)
    assert torch.equal(a, b)


def test_attn_extreme_scales_and_scores():
    """Scores far apart, values of very different sizes page by page, scales of zero."""
    g = gen_of(13)
    pool = random_pool(g, 2, 60, 2, 128, 16, [500, 300])
    pool.vs.copy_(torch.exp2(torch.randint(-60, 40, pool.vs.shape, generator=g, device="cuda").float()))
    pool.ks[:, ::5] = 0.0
    pool.vs[:, ::7] = 0.0
    q = torch.randn(3, 16, 128, generator=g, device="cuda").to(torch.bfloat16)
    seqs = [[0, 1, 499, 0], [1, 2, 250, 1]]
    check_attn(pool, q, seqs, scale=0.01)
    check_attn(pool, q * 0, seqs)
    pool.vs.fill_(0.0)
    o = check_attn(pool, q, seqs)
    assert bool((o[:3] == 0).all())


def test_attn_large_queries():
    """Queries near the ends of bf16's range take part with all their bits."""
    g = gen_of(14)
    pool = random_pool(g, 2, 10, 1, 64, 16, [150])
    q = torch.randn(2, 4, 64, generator=g, device="cuda")
    for by in (2.0 ** 60, 2.0 ** -60):
        check_attn(pool, (q * by).to(torch.bfloat16), [[0, 2, 140, 0]], scale=0.125 / by)
    mixed = (q * torch.exp2(torch.randint(-30, 1, (2, 4, 64), generator=g, device="cuda").float())).to(torch.bfloat16)
    check_attn(pool, mixed, [[0, 2, 140, 0]])


def test_attn_strides():
    g = gen_of(15)
    pool = random_pool(g, 2, 30, 2, 64, 32, [300, 200])
    wide = torch.randn(20, 3 * 8 * 64 + 8, generator=g, device="cuda").to(torch.bfloat16)
    q = wide[:, 512:1024].view(20, 8, 64)
    out = torch.full((20, 2 * 512), 5.0, dtype=torch.bfloat16, device="cuda")
    seqs = [[0, 1, 299, 0], [1, 18, 100, 1]]
    pool.attn(1, q, ints(seqs), out[:, 512:].view(20, 8, 64), max_rows=18)
    want, size = attn64(pool, 1, q, seqs, 0.125, 0)
    o = out[:, 512:].reshape(20, 8, 64)
    assert bool(((o.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size)[:19].all())
    assert bool((out[:, :512] == 5.0).all()) and bool((o[19] == 5.0).all())


def test_attn_offsets_beyond_32_bits():
    """A layer whose codes lie more than 2^32 bytes into the pool."""
    pages, kv, hd, page = 70000, 8, 128, 64
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 20 GB")
    shape = (1, pages, kv, page, hd)      # 4.6e9 codes
    k, v = (torch.empty(shape, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full(shape[:3], 2.0 ** -6, device="cuda") for _ in range(2))
    g = gen_of(16)
    ids = [pages - 1, 3, pages - 2, 65537, 69000]
    table = ints([ids, ids[::-1]])
    for i in ids:
        for t in (k, v):
            t[0, i] = torch.randint(-127, 128, shape[2:], generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    pool = P().PagePool(k, v, ks, vs, torch.ones(pages, dtype=torch.int32, device="cuda"), table, ints([320, 320]))
    q = torch.randn(24, 16, 128, generator=g, device="cuda").to(torch.bfloat16)
    check_attn(pool, q, [[0, 1, 319, 0], [1, 23, 290, 1]], layer=0)
    x = torch.randn(40, kv, hd, generator=g, device="cuda")
    pool.append(0, None, None, x, x, ints([[0, 40, 0, 0]]))
    kb, vb = torch.empty_like(x), torch.empty_like(x)
    pool.read(0, ints([[0, 40, 0, 0]]), kb, vb)
    assert torch.equal(kb, vb) and float((kb - x).abs().max()) <= float(pool.ks[0, ids[0]].max()) / 2


def test_attn_repeats_itself_and_serves_graphs():
    g = gen_of(17)
    pool = random_pool(g, 2, 400, 2, 128, 64, [5000, 300, 2000, 64])
    q = torch.randn(24, 16, 128, generator=g, device="cuda").to(torch.bfloat16)
    seqs = [[0, 1, 4999, 0], [1, 1, 299, 1], [2, 20, 1900, 2], [22, 1, 63, 3]]
    rows, o = ints(seqs), torch.zeros_like(q)
    first = check_attn(pool, q, seqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):      # on another stream than its tensors were made on
        pool.attn(1, q, rows, o, max_rows=20)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o[:23], first[:23])
    graphs = []
    for _ in range(2):      # two graphs that share the pool's work memory, replayed one behind the other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pool.attn(1, q, rows, o, max_rows=20)
            pool.attn(0, q, rows, o, max_rows=20)
            pool.attn(1, q, rows, o, max_rows=20)
        graphs.append(graph)
    for graph in graphs * 3:
        o.zero_()
        graph.replay()
        assert torch.equal(o[:23], first[:23])
    rows[0, 2], rows[2, 1] = 3000, 7      # other lengths, read on the device
    graphs[0].replay()
    seqs[0][2], seqs[2][1] = 3000, 7
    again = check_attn(pool, q, seqs)
    assert torch.equal(o[:9], again[:9])


def test_attn_many_sequences():
    g = gen_of(18)
    lens = [1 + (37 * i) % 90 for i in range(1500)]
    pool = random_pool(g, 2, sum(-(-n // 32) for n in lens), 1, 64, 32, lens)
    q = torch.randn(1500, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    check_attn(pool, q, [[i, 1, n - 1, i] for i, n in enumerate(lens)])


def test_attn_fewer_rows_than_a_descriptor_has():
    """max_rows bounds what is computed, also where a descriptor has more."""
    g = gen_of(19)
    pool = random_pool(g, 2, 10, 2, 64, 32, [200])
    q = torch.randn(30, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    o = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device="cuda")
    pool.attn(1, q, ints([[0, 30, 100, 0]]), o, max_rows=4)
    want, size = attn64(pool, 1, q, [[0, 30, 100, 0]], 0.125, 0)
    assert bool(((o.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size)[:4].all())
    assert bool((o[4:] == 5.0).all())


# ---- management against a plain model, request by request -------------------------------------------------------------------
class Model:
    def __init__(self, pages, page, sequences, max_pages):
        self.page, self.max = page, max_pages
        self.ref, self.table, self.len = [0] * pages, [[-1] * max_pages for _ in range(sequences)], [0] * sequences
        self.data = [None] * pages      # what a page holds: a mark

    def up(self, n):
        return -(-n // self.page)

    def extend(self, reqs):
        got, named, out, moves = [], set(), False, []
        for seq, n in reqs:
            if not 0 <= seq < len(self.len) or seq in named:
                got.append(0)
                continue
            named.add(seq)
            old = self.len[seq]
            n = max(n, old)
            if self.up(n) > self.max:
                got.append(0)
                continue
            last, part = old // self.page, n > old and old % self.page != 0
            copy = part and self.ref[self.table[seq][last]] > 1
            want = self.up(n) - self.up(old) + copy
            free = [i for i, r in enumerate(self.ref) if r == 0]
            if out or want > len(free):
                out = True
                got.append(0)
                continue
            if copy:
                a, b = self.table[seq][last], free.pop(0)
                moves.append((a, b))
                self.ref[a] -= 1
                self.ref[b] = 1
                self.table[seq][last] = b
            for j in range(self.up(old), self.up(n)):
                self.table[seq][j] = free.pop(0)
                self.ref[self.table[seq][j]], self.data[self.table[seq][j]] = 1, None
            self.len[seq] = n
            got.append(1)
        for a, b in moves:
            self.data[b] = self.data[a]
        return got

    def fork(self, forks):
        before, named = list(self.len), set()
        for src, dst, n, _ in forks:
            if not (0 <= src < len(before) and 0 <= dst < len(before)) or src == dst or dst in named:
                continue
            named.add(dst)
            if before[dst]:
                continue
            n = max(min(n, before[src]), 0)
            for j in range(self.up(n)):
                self.table[dst][j] = self.table[src][j]
                self.ref[self.table[src][j]] += 1
            self.len[dst] = n

    def trim(self, reqs):
        for seq, n in reqs:
            if not 0 <= seq < len(self.len):
                continue
            n = max(n, 0)
            for j in range(self.up(n), self.up(self.len[seq])):
                self.ref[self.table[seq][j]] -= 1
                self.table[seq][j] = -1
            self.len[seq] = min(self.len[seq], n)

    def compact(self):
        live = sum(r > 0 for r in self.ref)
        moves = list(zip([i for i, r in enumerate(self.ref) if r and i >= live], [i for i, r in enumerate(self.ref) if not r and i < live]))
        to = dict(moves)
        for a, b in moves:
            self.ref[b], self.ref[a], self.data[b] = self.ref[a], 0, self.data[a]
        self.table = [[to.get(i, i) for i in row] for row in self.table]


def same(pool, m):
    assert pool.ref.tolist() == m.ref and pool.length.tolist() == m.len and pool.table.tolist() == m.table
    used = [i for i, r in enumerate(m.ref) if r and m.data[i] is not None]
    for t, width in ((pool.k, 3), (pool.v, 3), (pool.ks, 1), (pool.vs, 1)):
        got = t[:, used].float().flatten(2)
        want = torch.tensor([[m.data[i]] for i in used], device="cuda", dtype=torch.float32)
        assert bool((got == want[None]).all()), width


def mark(pool, m, rng):
    """Every page in use that has no mark yet gets one, in all layers."""
    for i, r in enumerate(m.ref):
        if r and m.data[i] is None:
            m.data[i] = rng.randint(1, 127)
            for t in (pool.k, pool.v, pool.ks, pool.vs):
                t[:, i] = m.data[i]


@pytest.mark.parametrize("seed", range(6))
def test_management(seed):
    rng = random.Random(seed)
    page, pages, seqs, most = rng.choice([16, 32, 64, 128]), rng.choice([7, 60, 300, 5000]), 24, 12
    pool = P().PagePool.empty(rng.randint(1, 3), pages, rng.choice([1, 3]), rng.choice([64, 128]), page, seqs, most)
    m = Model(pages, page, seqs, most)
    for step in range(25):
        what = rng.choice(["extend", "extend", "extend", "fork", "fork", "trim", "compact"])
        n = rng.choice([1, 3, 24, 40])
        pick = lambda: rng.randint(-1, seqs)  # noqa: E731
        if what == "extend":
            reqs = [[pick(), rng.choice([0, -5, 1, page, page + 1, rng.randint(0, most * page), most * page + 1, 2 ** 31 - 1])] for _ in range(n)]
            got = torch.full((n,), 7, dtype=torch.int32, device="cuda")
            pool.extend(ints(reqs), got)
            assert got.tolist() == m.extend(reqs)
        elif what == "fork":
            forks = [[pick(), pick(), rng.choice([0, -3, rng.randint(0, most * page), 2 ** 31 - 1]), 0] for _ in range(n)]
            pool.fork(ints(forks))
            m.fork(forks)
        elif what == "trim":
            reqs = [[pick(), rng.choice([0, -2, rng.randint(0, most * page)])] for _ in range(n)]
            pool.trim(ints(reqs))
            m.trim(reqs)
        else:
            pool.compact()
            m.compact()
            assert pool.used() == sum(r > 0 for r in m.ref) and all(r > 0 for r in m.ref[:pool.used()])
        assert pool.ref.tolist() == m.ref and pool.length.tolist() == m.len and pool.table.tolist() == m.table, (step, what)


def test_management_moves_the_pages_contents():
    rng = random.Random(1)
    page, pool = 16, P().PagePool.empty(3, 50, 2, 64, 16, 10, 8)
    m = Model(50, page, 10, 8)
    for fn, arg in (("extend", [[i, 30 + 9 * i] for i in range(6)]), ("trim", [[1, 0], [3, 17]]), ("fork", [[0, 6, 25, 0], [0, 7, 20, 0], [4, 8, 66, 0], [4, 1, 64, 0]])):
        getattr(pool, fn)(ints(arg))
        getattr(m, fn)(arg)
        mark(pool, m, rng)
        same(pool, m)
    # page 1 of sequence 0 is partly used and shared by 0, 6 and 7: all three grow in one call, the last keeps it
    arg = [[6, 40], [0, 45], [8, 70], [7, 21]]
    pool.extend(ints(arg))
    assert m.extend(arg) == [1, 1, 1, 1]
    mark(pool, m, rng)
    same(pool, m)
    pool.trim(ints([[2, 0], [0, 0], [5, 1]]))
    m.trim([[2, 0], [0, 0], [5, 1]])
    pool.compact()
    m.compact()
    same(pool, m)
    used = pool.used()
    pool.copy(ints([[0, used], [1, used + 1], [-1, used + 2], [2, 50], [3, 3]]))
    for t in (pool.k, pool.v, pool.ks, pool.vs):
        assert torch.equal(t[:, 0], t[:, used]) and torch.equal(t[:, 1], t[:, used + 1])
    same(pool, m)


def test_management_large_pool():
    """More pages than a block looks at in one round, large pages, and a request list of full length."""
    pool = P().PagePool.empty(1, 30000, 8, 128, 128, 1024, 29)
    m = Model(30000, 128, 1024, 29)
    reqs = [[i, 1 + (i * 331) % 3712] for i in range(1024)]
    got = torch.zeros(1024, dtype=torch.int32, device="cuda")
    pool.extend(ints(reqs), got)
    assert got.tolist() == m.extend(reqs)
    drop = [[i, 0] for i in range(0, 1024, 3)]
    pool.trim(ints(drop))
    m.trim(drop)
    pool.compact()
    m.compact()
    assert pool.ref.tolist() == m.ref and pool.table.tolist() == m.table
    pool.trim(ints([[i % 1024, 5] for i in range(1024)]))
    m.trim([[i, 5] for i in range(1024)])
    assert pool.ref.tolist() == m.ref and pool.length.tolist() == m.len


# ---- a run of them together ---------------------------------------------------------------------------------------------------
def test_a_run_of_all_of_them():
    """Two prompts in chunks, a fork, decode steps of all three, a rollback, a compaction: attention against 64-bit sums over what
    the cache holds, and what it holds against what was stored."""
    g = gen_of(21)
    kv, hd, page, heads, layers = 2, 64, 16, 8, 2
    pool = P().PagePool.empty(layers, 80, kv, hd, page, 4, 20)
    inv, factor = P().rope_freqs(hd // 2, 1e4, P().ROPE_PARTS, 4.0, 256)
    r = P().Rope(torch.from_numpy(inv).cuda(), interleaved=True, factor=factor)
    stored = {s: [torch.zeros(0, kv, hd, dtype=torch.float64, device="cuda")] * 2 for s in range(3)}

    def step(rows):      # [(rows, sequence)]
        desc, row, grow = [], 0, []
        for n, s in rows:
            desc.append([row, n, stored[s][0].shape[0], s])
            grow.append([s, stored[s][0].shape[0] + n])
            row += n
        pool.extend(ints(grow))
        for layer in range(layers):
            q, k, v = (torch.randn(row, n, hd, generator=g, device="cuda").to(torch.bfloat16).float() for n in (heads, kv, kv))
            q2, o = torch.empty_like(q), torch.empty(row, heads, hd, dtype=torch.bfloat16, device="cuda")
            pool.append(layer, r, q, k, v, ints(desc), q2, rounded=True)
            pool.attn(layer, q2, ints(desc), o, max_rows=max(n for n, _ in rows))
            want, size = attn64(pool, layer, q2, desc, hd ** -0.5, 0)
            assert bool(((o.double() - want).abs() <= BF16 * want.abs() + (1 + BF16) * WEIGHTS * size).all())
            if layer == layers - 1:
                for row0, n, p, s in desc:
                    pos = torch.arange(p, p + n, device="cuda")
                    kr = turned(k[row0:row0 + n], pos, r.inv, True, factor)[0]
                    stored[s] = [torch.cat([stored[s][0], kr]), torch.cat([stored[s][1], v[row0:row0 + n].double()])]
                    for got, x in zip(held(pool, layer, s, p + n), stored[s]):
                        top = x.abs().max()      # steps of at most top / 63.5, a page's codes rounded a few times: each half a step of the scale then
                        assert float((got - x).abs().max()) <= 1.5 * float(top) / 63.5

    step([(37, 0), (50, 1)])
    step([(20, 0), (1, 1)])
    pool.fork(ints([[0, 2, 57, 0]]))
    stored[2] = list(stored[0])
    for _ in range(20):
        step([(1, 0), (1, 1), (1, 2)])
    step([(4, 2), (4, 0)])
    pool.trim(ints([[2, 60], [1, 0]]))      # a rollback of drafted tokens, and a sequence that ended
    stored[2] = [x[:60] for x in stored[2]]
    stored[1] = [x[:0] for x in stored[1]]
    pool.compact()
    for _ in range(3):
        step([(1, 2), (1, 0)])
    step([(70, 1), (1, 0)])
    pool.trim(ints([[s, 0] for s in range(4)]))
    assert pool.used() == 0 and bool((pool.table == -1).all())


def test_wrapper_refusals():
    pool = P().PagePool.empty(1, 4, 2, 64, 16, 2, 2)
    x, rows = torch.zeros(3, 2, 64, device="cuda"), ints([[0, 3, 0, 0]])
    bad = [lambda: pool.append(0, None, None, x[:, :1], x, rows), lambda: pool.append(0, None, None, x, x.double(), rows), lambda: pool.append(1, None, None, x, x, rows),
           lambda: pool.append(0, None, None, x, x, rows.long()), lambda: pool.append(0, None, None, x, x, rows.cpu()), lambda: pool.attn(0, x, rows, x[:2], max_rows=3),
           lambda: pool.attn(0, x, rows, x, max_rows=3, work=rows.flatten()), lambda: pool.attn(0, x[:, :, ::2], rows, x, max_rows=3), lambda: pool.read(0, rows, x, x[:2]),
           lambda: pool.extend(ints([1, 2])), lambda: pool.extend(ints([[0, 1]] * 3), ints([0])), lambda: pool.fork(ints([[0, 1]])), lambda: pool.extend(ints([[0, 0]] * 1025)),
           lambda: P().PagePool(pool.k, pool.v, pool.ks, pool.vs, pool.ref[:3], pool.table, pool.length), lambda: P().Rope(torch.zeros(4, device="cuda").double()),
           lambda: P().rope(P().Rope(inv_of(64)), x, None, ints([1, 2])), lambda: P().PagePool.empty(1, 4, 2, 96, 16, 2, 2).compact()]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()


def decode_run(pool, steps, wait, seed):
    """Store and attend `steps` tokens of three sequences, each step's queries made from the last one's results."""
    g = gen_of(seed)
    r = P().Rope(inv_of(64))
    q = torch.randn(3, 8, 64, generator=g, device="cuda").to(torch.bfloat16)
    kv = torch.randn(steps, 2, 3, 2, 64, generator=g, device="cuda").to(torch.bfloat16)
    rows = [ints([[0, 1, 40 + i, 0], [1, 1, 7 + i, 1], [2, 1, 100 + i, 2]]) for i in range(steps)]
    grow = [ints([[0, 41 + i], [1, 8 + i], [2, 101 + i]]) for i in range(steps)]
    outs = [torch.empty_like(q) for _ in range(steps)]
    turned_q = torch.empty_like(q)
    for i in range(steps):
        pool.extend(grow[i])
        pool.append(0, r, q if i == 0 else outs[i - 1], kv[i, 0], kv[i, 1], rows[i], turned_q)
        pool.attn(0, turned_q, rows[i], outs[i], max_rows=1)
        if wait:
            torch.cuda.synchronize()
    torch.cuda.synchronize()
    return torch.stack(outs)


def test_steps_queued_one_behind_the_other():
    """Calls that start before their predecessors have ended, whose inputs these write (codes that are then fetched by bulk copies, queries, tables),
    give what the same calls give one by one, as dependent launches and as ordinary ones."""
    lib = P().L.load()
    got = []
    for wait, mode in ((True, -1), (False, -1), (False, 0), (False, 1)):
        pool = P().PagePool.empty(1, 60, 2, 64, 16, 3, 12)
        for t in (pool.k, pool.v):
            t.zero_()
        for t in (pool.ks, pool.vs):
            t.fill_(2.0 ** -6)
        pool.extend(ints([[0, 40], [1, 7], [2, 100]]))
        lib.nsl_dependent_launch(mode)
        try:
            got.append(decode_run(pool, 40, wait, 31))
        finally:
            lib.nsl_dependent_launch(-1)
    assert all(torch.equal(got[0], x) for x in got[1:])
    assert bool(torch.isfinite(got[0]).all()) and lib.nsl_pages_attn_status() == 0


def test_two_calls_beside_one_another():
    """Two streams, each with work memory of its own: both give what a call alone gives; few rows and many."""
    g = gen_of(41)
    pool = random_pool(g, 2, 700, 2, 128, 16, [3000, 2000, 700])
    calls = []
    for seqs in ([[0, 1, 2999, 0], [1, 1, 1999, 1]], [[0, 150, 550, 2], [150, 3, 1900, 1]]):
        q = torch.randn(153, 16, 128, generator=g, device="cuda").to(torch.bfloat16)
        calls.append((q, ints(seqs), max(n for _, n, _, _ in seqs), torch.empty_like(pool.attn_work), torch.cuda.Stream(), [torch.zeros_like(q) for _ in range(8)], torch.zeros_like(q)))
    for q, rows, most, work, _, _, alone in calls:
        pool.attn(1, q, rows, alone, max_rows=most)
    torch.cuda.synchronize()
    for i in range(8):
        for q, rows, most, work, stream, outs, _ in calls:
            with torch.cuda.stream(stream):
                pool.attn(1, q, rows, outs[i], max_rows=most, work=work)
    torch.cuda.synchronize()
    for *_, outs, alone in calls:
        assert all(torch.equal(o, alone) for o in outs)


def test_attn_a_sequence_in_several_descriptors():
    g = gen_of(43)
    pool = random_pool(g, 2, 20, 2, 64, 64, [900])
    q = torch.randn(5, 8, 64, generator=g, device="cuda").to(torch.bfloat16)
    check_attn(pool, q, [[0, 1, 899, 0], [1, 3, 500, 0], [4, 1, 3, 0]])
    check_attn(pool, q, [[0, 1, 899, 0], [1, 1, 500, 0], [4, 1, 899, 0]])


@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_attn_scales_of_either_sign(scale):
    g = gen_of(44)
    pool = random_pool(g, 2, 20, 2, 64, 64, [700])
    q = torch.randn(70, 8, 64, generator=g, device="cuda").to(torch.bfloat16)
    check_attn(pool, q, [[0, 1, 699, 0]], scale=scale)
    check_attn(pool, q, [[0, 70, 600, 0]], scale=scale)
