"""The paged cache's host side: what its calls refuse (nothing is launched, no GPU is needed), and the rotary frequency tables."""
import ctypes as C
import math

import numpy as np
import pytest

from nanoseedlm_b200 import lib as L
from nanoseedlm_b200 import pages as P

A = C.c_void_p(0x10000)      # an address that is never followed: the call is refused before
ODD = C.c_void_p(0x10008)


def pool(**kw):
    f = dict(k=0x10000, v=0x10000, ks=0x10000, vs=0x10000, ref=0x10000, table=0x10000, len=0x10000, work=0x10000, n_layer=2, n_pages=8, n_kv=2, hd=128, page=64, n_seq=4, max_pages=4, pad=0)
    f.update(kw)
    return L.NslPages(*(f[n] for n, _ in L.NslPages._fields_))


def rope(**kw):
    f = dict(inv=0x10000, rot=128, layout=0, factor=1.0, pad=0)
    f.update(kw)
    return L.NslRope(*(f[n] for n, _ in L.NslRope._fields_))


def refused(fn, *args):
    lib = L.load()
    lib.nsl_last_error()
    before = lib.nsl_launch_count()
    getattr(lib, fn)(None, *args)
    assert L.last_error().startswith(fn), args
    assert lib.nsl_launch_count() == before


BAD_POOLS = [dict(k=0), dict(vs=0), dict(table=0), dict(work=0), dict(k=0x10008), dict(n_layer=0), dict(n_pages=0), dict(n_pages=(1 << 20) + 1), dict(n_kv=0), dict(n_kv=1025), dict(hd=96), dict(hd=256),
             dict(page=8), dict(page=48), dict(page=256), dict(n_seq=0), dict(max_pages=0), dict(max_pages=1 << 25)]


@pytest.mark.parametrize("bad", BAD_POOLS, ids=str)
def test_pools_that_are_refused(bad):
    p = C.byref(pool(**bad))
    refused("nsl_pages_append", p, 0, rope(rot=64), 1, A, 2048, A, 2048, 16, A, 256, A, 256, A, 1, 4)
    refused("nsl_pages_read", p, 0, 1, A, 256, A, 256, A, 1, 4)
    refused("nsl_pages_attn", p, 0, 1, A, 2048, 16, 0.1, 0, A, 1, 4, 4, 1, A, 2048, A)
    refused("nsl_pages_extend", p, A, 1, None)
    refused("nsl_pages_fork", p, A, 1)
    refused("nsl_pages_trim", p, A, 1)
    refused("nsl_pages_compact", p)
    refused("nsl_pages_copy", p, A, 1)


@pytest.mark.parametrize("kw", [dict(layer=2), dict(layer=-1), dict(type=3), dict(rope=rope(rot=8)), dict(rope=rope(rot=144)), dict(rope=rope(rot=-16)), dict(rope=rope(inv=0)), dict(rope=rope(layout=2)),
                                dict(q=None), dict(q=ODD), dict(qs=2047), dict(qs=2052), dict(qo=None), dict(n_head=-1), dict(k=None), dict(k=ODD), dict(ks=255), dict(v=None), dict(vs=260),
                                dict(seqs=None)], ids=lambda kw: ",".join(kw))
def test_append_refusals(kw):
    f = dict(layer=0, rope=rope(), type=1, q=A, qs=2048, qo=A, qos=2048, n_head=16, k=A, ks=256, v=A, vs=256, seqs=A, n=1, T=4)
    f.update(kw)
    refused("nsl_pages_append", C.byref(pool()), *(f[n] for n in ("layer", "rope", "type", "q", "qs", "qo", "qos", "n_head", "k", "ks", "v", "vs", "seqs", "n", "T")))


@pytest.mark.parametrize("kw", [dict(layer=2), dict(type=-1), dict(k=None), dict(v=ODD), dict(ks=128), dict(seqs=None)], ids=lambda kw: ",".join(kw))
def test_read_refusals(kw):
    f = dict(layer=0, type=0, k=A, ks=256, v=A, vs=256, seqs=A, n=1, T=4)
    f.update(kw)
    refused("nsl_pages_read", C.byref(pool()), *(f[n] for n in ("layer", "type", "k", "ks", "v", "vs", "seqs", "n", "T")))


@pytest.mark.parametrize("kw", [dict(layer=2), dict(qt=5), dict(ot=0), dict(ot=3), dict(n_head=0), dict(n_head=15), dict(q=None), dict(q=ODD), dict(qs=2044), dict(o=None), dict(os=1024), dict(seqs=None), dict(n=4097),
                                dict(work=None), dict(work=ODD)], ids=lambda kw: ",".join(kw))
def test_attn_refusals(kw):
    f = dict(layer=0, qt=1, q=A, qs=2048, n_head=16, scale=0.1, window=0, seqs=A, n=1, max_rows=4, T=4, ot=1, o=A, os=2048, work=A)
    f.update(kw)
    refused("nsl_pages_attn", C.byref(pool()), *(f[n] for n in ("layer", "qt", "q", "qs", "n_head", "scale", "window", "seqs", "n", "max_rows", "T", "ot", "o", "os", "work")))


@pytest.mark.parametrize("kw", [dict(type=7), dict(hd=24), dict(hd=528), dict(q=ODD), dict(q=None), dict(qs=2040), dict(ko=None), dict(pos=None), dict(n_head=0, n_kv=0), dict(r=rope(rot=0)), dict(r=rope(rot=136))],
                         ids=lambda kw: ",".join(kw))
def test_rope_refusals(kw):
    f = dict(r=rope(), type=1, hd=128, q=A, qs=2048, qo=A, qos=2048, n_head=16, k=A, ks=256, ko=A, kos=256, n_kv=2, pos=A, T=3)
    f.update(kw)
    refused("nsl_rope", *(f[n] for n in ("r", "type", "hd", "q", "qs", "qo", "qos", "n_head", "k", "ks", "ko", "kos", "n_kv", "pos", "T")))


def test_lists_that_are_refused():
    p = C.byref(pool())
    for fn, more in (("nsl_pages_extend", (None,)), ("nsl_pages_fork", ()), ("nsl_pages_trim", ())):
        refused(fn, p, A, 1025, *more)
        refused(fn, p, None, 1, *more)
    refused("nsl_pages_copy", p, None, 1)


def test_empty_calls_do_nothing():
    lib, p = L.load(), C.byref(pool())
    lib.nsl_last_error()
    before = lib.nsl_launch_count()
    lib.nsl_pages_append(None, p, 0, rope(), 1, A, 2048, A, 2048, 16, A, 256, A, 256, A, 0, 4)
    lib.nsl_pages_append(None, p, 0, rope(), 1, A, 2048, A, 2048, 16, A, 256, A, 256, A, 1, 0)
    lib.nsl_pages_read(None, p, 0, 1, A, 256, A, 256, A, 0, 4)
    lib.nsl_pages_attn(None, p, 0, 1, A, 2048, 16, 0.1, 0, A, 0, 4, 4, 1, A, 2048, A)
    lib.nsl_pages_attn(None, p, 0, 1, A, 2048, 16, 0.1, 0, A, 1, 0, 4, 1, A, 2048, A)
    lib.nsl_rope(None, rope(), 1, 128, A, 2048, A, 2048, 16, A, 256, A, 256, 2, A, 0)
    for fn in (lib.nsl_pages_fork, lib.nsl_pages_trim, lib.nsl_pages_copy):
        fn(None, p, A, 0)
    lib.nsl_pages_extend(None, p, A, 0, None)
    assert L.last_error() == "" and lib.nsl_launch_count() == before


# ---- frequencies: float32 of the formulas in 64 bits, so they agree to half a step (2^-24) and the order of the operations ------
def expected(kind, rot, theta, scale, ctx, fast, slow):
    p = np.arange(rot // 2, dtype=np.float64)
    f = theta ** (-2 * p / rot)
    if kind == P.ROPE_LINEAR:
        return f / scale, 1.0
    if kind == P.ROPE_BASE:
        return (theta * scale ** (rot / (rot - 2))) ** (-2 * p / rot), 1.0
    if kind == P.ROPE_PARTS:
        turns = lambda beta: rot * math.log(ctx / (beta * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(turns(fast)), 0), min(math.ceil(turns(slow)), rot - 1)
        hi = hi if hi > lo else lo + 0.001
        keep = 1 - np.clip((p - lo) / (hi - lo), 0, 1)
        return f / scale * (1 - keep) + f * keep, 0.1 * math.log(scale) + 1
    return f, 1.0


@pytest.mark.parametrize("rot", [16, 64, 128, 256])
@pytest.mark.parametrize("kind,scale,ctx", [(P.ROPE_PLAIN, 1.0, 0), (P.ROPE_LINEAR, 4.0, 0), (P.ROPE_BASE, 8.0, 0), (P.ROPE_PARTS, 4.0, 32768), (P.ROPE_PARTS, 1.0, 4096), (P.ROPE_PARTS, 40.0, 4096)])
@pytest.mark.parametrize("theta", [1e4, 1e6])
def test_frequencies(rot, kind, scale, ctx, theta):
    inv, factor = P.rope_freqs(rot, theta, kind, scale, ctx)
    want, f = expected(kind, rot, theta, scale, ctx, 32.0, 1.0)
    assert np.all(np.abs(inv - want) <= 2.0 ** -24 * want * (1 + 1e-6) + 1e-14 * want)
    assert abs(factor - f) <= 2.0 ** -24 * f
    if kind == P.ROPE_BASE:      # the two ends: kept, and divided by scale
        assert inv[0] == 1.0 and abs(inv[-1] * scale / theta ** (-(rot - 2) / rot) - 1) < 1e-6


@pytest.mark.parametrize("args", [(64, 1.0), (63, 1e4), (0, 1e4), (64, 1e4, 7), (64, 1e4, P.ROPE_LINEAR, 0.5), (64, 1e4, P.ROPE_PARTS, 4.0, 0), (64, 1e4, P.ROPE_PARTS, 4.0, 4096, 1.0, 32.0), (2, 1e4, P.ROPE_BASE, 2.0),
                                  (64, float("nan")), (64, 1e4, P.ROPE_LINEAR, float("nan"))], ids=str)
def test_frequency_refusals(args):
    L.load().nsl_last_error()
    with pytest.raises(ValueError):
        P.rope_freqs(*args)
