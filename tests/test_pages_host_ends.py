"""More of what the paged cache's calls refuse on the host (nothing is launched, no GPU is needed)."""
import ctypes as C
import threading

import pytest
from test_pages_host import A, pool, rope

from nanoseedlm_b200 import lib as L
from nanoseedlm_b200 import pages as P


def refused(why, fn, *args):
    lib = L.load()
    lib.nsl_last_error()
    before = lib.nsl_launch_count()
    getattr(lib, fn)(None, *args)
    msg = L.last_error()
    assert msg.startswith(fn) and why in msg, (msg, args)
    assert lib.nsl_launch_count() == before


# ---- outputs that overlap inputs or one another ----------------------------------------------------------------------------
def at(byte):
    return C.c_void_p(0x10000 + byte)


W = 2 * 1024      # bytes of a row of 16 x 64 bf16 values
OVERLAPS = [  # (output's first byte, its stride in values): inputs start at 0, 8 rows of 1024 bf16 values in rows of 4096 bytes
    (16, 2048), (W - 16, 2048), (4096 - W + 16, 2048), (7 * 4096, 2048), (-7 * 4096, 2048), (0, 4096), (2 * 4096, 1024), (4096 * 3 + 2032, 2048), (W, 1536)]


@pytest.mark.parametrize("byte,stride", OVERLAPS)
def test_outputs_that_overlap(byte, stride):
    p = C.byref(pool(hd=64, n_kv=16))
    q = at(0x100000)
    o = at(0x100000 + byte)
    far = at(0x900000)
    refused("overlap", "nsl_pages_attn", p, 0, 1, q, 2048, 16, 0.1, 0, A, 1, 4, 8, 1, o, stride, A)
    refused("overlap", "nsl_rope", rope(rot=64), 1, 64, q, 2048, o, stride, 16, None, 0, None, 0, 0, A, 8)
    refused("overlap", "nsl_rope", rope(rot=64), 1, 64, q, 2048, q, 2048, 16, far, 2048, o, stride, 16, A, 8)
    refused("overlap", "nsl_rope", rope(rot=64), 1, 64, far, 2048, o, stride, 16, q, 2048, q, 2048, 16, A, 8)
    refused("overlap", "nsl_pages_append", p, 0, rope(rot=64), 1, q, 2048, o, stride, 16, far, 2048, far, 2048, A, 1, 8)
    refused("overlap", "nsl_pages_append", p, 0, rope(rot=64), 1, far, 2048, o, stride, 16, q, 2048, at(0xF00000), 2048, A, 1, 8)
    refused("overlap", "nsl_pages_append", p, 0, rope(rot=64), 1, far, 2048, o, stride, 16, at(0xF00000), 2048, q, 2048, A, 1, 8)
    refused("overlap", "nsl_pages_read", p, 0, 1, q, 2048, o, stride, A, 1, 8)


def test_outputs_of_another_width_that_overlap():
    refused("overlap", "nsl_pages_attn", C.byref(pool()), 0, 0, at(0), 2048, 16, 0.1, 0, A, 1, 4, 8, 1, at(4096), 2048, A)      # f32 rows of 8192 bytes, bf16 results within them


# ---- whose refusal a call reports -------------------------------------------------------------------------------------------------
def test_a_call_reports_its_own_refusal_only():
    lib, p = L.load(), C.byref(pool())
    lib.nsl_last_error()
    lib.nsl_pages_fork(None, p, None, 1)      # refused, and not read
    lib.nsl_pages_copy(None, p, A, 0)         # an empty call
    assert lib.nsl_pages_error() == b""
    with pytest.raises(ValueError, match="nsl_rope_freqs"):
        P.rope_freqs(63, 1e4)
    P.rope_freqs(64, 1e4)
    assert lib.nsl_pages_error() == b""
    assert L.last_error().startswith("nsl_pages_fork") and L.last_error() == ""
    lib.nsl_pages_trim(None, p, None, 1)
    assert lib.nsl_pages_error().startswith(b"nsl_pages_trim") and L.last_error() == ""      # read here, read there


def test_a_call_reports_nothing_of_other_threads():
    lib, p = L.load(), C.byref(pool())
    lib.nsl_last_error()
    lib.nsl_pages_copy(None, p, A, 0)
    seen = []
    t = threading.Thread(target=lambda: (lib.nsl_pages_fork(None, p, None, 1), seen.append(lib.nsl_pages_error())))
    t.start()
    t.join()
    assert seen[0].startswith(b"nsl_pages_fork") and lib.nsl_pages_error() == b""
    lib.nsl_last_error()


# ---- frequencies by parts: known values, worked out apart from the code (40 decimal digits), to half a step of float32 (2^-24) -----------
@pytest.mark.parametrize("rot,scale,factor,values", [
    (128, 16.0, 1.277258872223978, {0: 1.0, 10: 2.371373705661655e-1, 20: 5.623413251903491e-2, 21: 4.694085999795940e-2, 33: 4.600435467850347e-3, 45: 1.517716047318249e-4,
                                    46: 8.334508951020775e-5, 63: 7.217387404309114e-6}),      # pairs 20.94 and 45.03: the ramp from 20 to 46
    (64, 40.0, 1.368887945411394, {0: 1.0, 10: 5.623413251903491e-2, 11: 3.900692656714386e-2, 16: 5.5e-3, 22: 1.778279410038923e-4, 23: 3.333803580408310e-5,
                                   31: 3.333803580408310e-6})])                                # pairs 10.47 and 22.51: from 10 to 23
def test_known_frequencies_by_parts(rot, scale, factor, values):
    inv, f = P.rope_freqs(rot, 1e4, P.ROPE_PARTS, scale, 4096)
    assert abs(f - factor) <= 2.0 ** -24 * factor * 1.001
    for p, want in values.items():
        assert abs(float(inv[p]) - want) <= 2.0 ** -24 * want * 1.001, p


@pytest.mark.parametrize("args", [(64, float("inf")), (64, 1e4, P.ROPE_LINEAR, float("inf")), (64, 1e4, P.ROPE_BASE, float("inf")), (64, 1e4, P.ROPE_PARTS, float("inf"), 4096)], ids=str)
def test_frequencies_of_infinite_arguments(args):
    with pytest.raises(ValueError, match="nsl_rope_freqs"):
        P.rope_freqs(*args)


def test_a_status_that_cannot_be_read_is_an_error():
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is a device to read")
    L.load().nsl_last_error()
    assert L.load().nsl_pages_attn_status() == -1
    assert b"nsl_pages_attn_status" in L.load().nsl_pages_error() and L.last_error() == ""
