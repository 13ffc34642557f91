"""Python handle of the paged 8-bit KV cache and its operators (include/nslm_pages.h): rotary positions, the store into pages,
attention over them, and the pages' management.  torch supplies device memory and streams; every call goes to the library and
only enqueues work on the current stream."""
import ctypes as C

import numpy as np
import torch

from . import lib as L

NSL_F32, NSL_BF16, NSL_F32_BF16 = 0, 1, 2
ROPE_PLAIN, ROPE_LINEAR, ROPE_BASE, ROPE_PARTS = 0, 1, 2, 3


def rope_freqs(rot, theta, kind=ROPE_PLAIN, scale=1.0, ctx=0, beta_fast=32.0, beta_slow=1.0):
    """-> (frequencies float32 [rot / 2] on the host, factor): see nsl_rope_freqs."""
    inv, factor = np.zeros(max(rot // 2, 1), np.float32), C.c_float()
    if L.load().nsl_rope_freqs(kind, rot, theta, scale, ctx, beta_fast, beta_slow, C.c_void_p(inv.ctypes.data), C.byref(factor)):
        _done()
    return inv, factor.value


class Rope:
    """How heads are rotated: inv [rot / 2] (float32, device) angles per position, half or interleaved pairs, a factor on the result."""

    def __init__(self, inv, interleaved=False, factor=1.0):
        if inv.dtype != torch.float32 or not inv.is_cuda or not inv.is_contiguous() or inv.dim() != 1:
            raise ValueError("inv: a contiguous float32 device vector")
        self.inv = inv
        self.struct = L.NslRope(inv.data_ptr(), 2 * inv.numel(), int(interleaved), factor, 0)


_NO_ROPE = L.NslRope(0, 0, 0, 1.0, 0)


_TYPES = {torch.bfloat16: (NSL_BF16, NSL_BF16), torch.float32: (NSL_F32, NSL_F32_BF16)}


def _type(t, rounded=False):
    try:
        return _TYPES[t.dtype][rounded]
    except KeyError:
        raise ValueError(f"{t.dtype}: float32 or bfloat16 rows") from None


def _rows(t, name, like=None):
    """[T][heads][hd] with dense heads: the row stride in elements."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name}: [T][heads][hd], got {tuple(shape)}")
    T, heads, hd = shape
    rs, hs, es = t.stride()
    if es != 1 or (hs != hd and heads > 1):
        raise ValueError(f"{name}: dense heads, got strides {t.stride()}")
    if like is not None and like is not t:
        other = like.shape
        if T != other[0] or hd != other[2] or t.dtype != like.dtype:
            raise ValueError(f"{name}: another type, number of rows or head width than the other rows")
    return rs if T > 1 else heads * hd


def _ints(t, name, width):
    """A contiguous int32 list [n][width] ([n] for width 0): n."""
    shape = t.shape
    if t.dtype != torch.int32 or not t.is_contiguous() or (len(shape) != 2 or shape[1] != width if width else len(shape) != 1):
        raise ValueError(f"{name}: a contiguous int32 tensor {'[n][%d]' % width if width else '[n]'}")
    return shape[0]


_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _here(index, *tensors):
    """All on the device `index`, and that the current one."""
    if index < 0 or index != _device():
        raise ValueError(f"tensors on {f'cuda:{index}' if index >= 0 else 'the host'}, but the current device is cuda:{torch.cuda.current_device()}")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"a tensor on {t.device} among tensors on cuda:{index}")


def _done():
    """Raises what this thread's last call was refused for."""
    msg = L.load().nsl_pages_error()
    if msg:
        raise ValueError(msg.decode())


# The stream's handle without a Stream object around it (a microsecond a call), where torch offers that.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


def _ptr(t):
    return t.data_ptr() if t is not None else None


def rope(r, q, k, pos, q_out=None, k_out=None, rounded=False):
    """Rotates the heads of q [T][heads][hd] and k (or None) at positions pos (int32 [T]); in place without outputs.  rounded: float32
    results are rounded to bf16."""
    q_out, k_out = q if q_out is None else q_out, k if k_out is None else k_out
    index = q.get_device()
    _here(index, k, pos, q_out, k_out, r.inv)
    qs, (T, heads, hd) = _rows(q, "q"), q.shape
    qos = qs
    if q_out is not q:
        qos = _rows(q_out, "q_out", q)
        if q_out.shape[1] != heads:
            raise ValueError("q_out: the shape of q")
    if _ints(pos, "pos", 0) != T:
        raise ValueError("pos: one position a row")
    ks = kos = kv = 0
    if k is not None:
        ks = kos = _rows(k, "k", q)
        kv = k.shape[1]
        if k_out is not k:
            kos = _rows(k_out, "k_out", q)
            if k_out.shape[1] != kv:
                raise ValueError("k_out: the shape of k")
    L.load().nsl_rope(_stream(index), r.struct, _type(q, rounded), hd, _ptr(q), qs, _ptr(q_out), qos, heads, _ptr(k), ks, _ptr(k_out), kos, kv, _ptr(pos), T)
    _done()


def seq_rows(rows, device="cuda"):
    """Descriptors [(first row, rows, position of the first, sequence)] as the device list that the calls take."""
    return torch.tensor(rows, dtype=torch.int32, device=device).reshape(-1, 4)


class PagePool:
    def __init__(self, k, v, ks, vs, ref, table, length):
        """k, v: int8 [layers][pages][kv heads][page][hd]; ks, vs: float32 [layers][pages][kv heads]; ref: int32 [pages]; table: int32
        [sequences][pages of a sequence], -1 where there is none; length: int32 [sequences]."""
        shape, device = k.shape, k.device
        for t, dt, sh, name in ((k, torch.int8, shape, "k"), (v, torch.int8, shape, "v"), (ks, torch.float32, shape[:3], "ks"), (vs, torch.float32, shape[:3], "vs"),
                                (ref, torch.int32, shape[1:2], "ref"), (table, torch.int32, table.shape, "table"), (length, torch.int32, table.shape[:1], "length")):
            if t.dtype != dt or t.shape != sh or not t.is_contiguous() or t.device != device or not t.is_cuda:
                raise ValueError(f"{name}: a contiguous {dt} device tensor {tuple(sh)} on {device}, got {t.dtype} {tuple(t.shape)}")
        if k.dim() != 5 or table.dim() != 2:
            raise ValueError("k: [layers][pages][kv heads][page][hd]; table: [sequences][pages of a sequence]")
        self.lib, self.device, self.index = L.load(), device, device.index
        self.k, self.v, self.ks, self.vs, self.ref, self.table, self.length = k, v, ks, vs, ref, table, length
        self.work = torch.empty(4 + 3 * shape[1], dtype=torch.int32, device=device)
        self.attn_work = torch.empty(self.lib.nsl_pages_attn_work() // 4, dtype=torch.int32, device=device)
        self.kv, self.hd, self.page = shape[2], shape[4], shape[3]
        self.struct = L.NslPages(*(t.data_ptr() for t in (k, v, ks, vs, ref, table, length, self.work)), shape[0], shape[1], shape[2], shape[4], shape[3], table.shape[0],
                               table.shape[1], 0)
        self._p = C.byref(self.struct)
        self._works = {_stream(self.index): self.attn_work}      # by stream: calls on one run one behind the other

    def _work_of(self, stream):
        """Attention's work memory: the stream's own, made at its first call; in a capture the graph's, from the capture's memory."""
        if stream and _capturing():      # (the default stream, 0, is never captured)
            return torch.empty_like(self.attn_work)
        work = self._works.get(stream)
        if work is None:
            work = self._works[stream] = torch.empty_like(self.attn_work)
        return work

    @classmethod
    def empty(cls, layers, pages, kv, hd, page, sequences, max_pages, device="cuda"):
        """A pool without sequences.  Its codes and scales are not cleared: what is read has been written."""
        codes = lambda: torch.empty((layers, pages, kv, page, hd), dtype=torch.int8, device=device)  # noqa: E731
        scales = lambda: torch.empty((layers, pages, kv), dtype=torch.float32, device=device)  # noqa: E731
        return cls(codes(), codes(), scales(), scales(), torch.zeros(pages, dtype=torch.int32, device=device),
                   torch.full((sequences, max_pages), -1, dtype=torch.int32, device=device), torch.zeros(sequences, dtype=torch.int32, device=device))

    def append(self, layer, r, q, k, v, rows, q_out=None, rounded=False):
        """Rotates q (or None; in place without q_out) and k as r says (None: not at all) and stores k, v [T][kv heads][hd] at the
        descriptors' positions."""
        _here(self.index, q, k, v, rows, q_out, r.inv if r is not None else None)
        q_out = q if q_out is None else q_out
        ks, vs, shape = _rows(k, "k"), _rows(v, "v", k), k.shape
        T = shape[0]
        if shape[1] != self.kv or shape[2] != self.hd or v.shape[1] != self.kv:
            raise ValueError(f"k, v: [T][{self.kv}][{self.hd}]")
        qs = qos = heads = 0
        if q is not None:
            qs = qos = _rows(q, "q", k)
            heads = q.shape[1]
            if q_out is not q:
                qos = _rows(q_out, "q_out", k)
                if q_out.shape[1] != heads:
                    raise ValueError("q_out: the shape of q")
        n = _ints(rows, "rows", 4)
        self.lib.nsl_pages_append(_stream(self.index), self._p, layer, r.struct if r is not None else _NO_ROPE, _type(k, rounded), _ptr(q), qs, _ptr(q_out), qos, heads, _ptr(k), ks, _ptr(v), vs,
                                  _ptr(rows), n, T)
        _done()

    def read(self, layer, rows, k_out, v_out, rounded=False):
        """The values at the descriptors' positions -> k_out, v_out [T][kv heads][hd]."""
        _here(self.index, rows, k_out, v_out)
        ks, vs = _rows(k_out, "k_out"), _rows(v_out, "v_out", k_out)
        shape = k_out.shape
        if shape[1] != self.kv or shape[2] != self.hd or v_out.shape[1] != self.kv:
            raise ValueError(f"k_out, v_out: [T][{self.kv}][{self.hd}]")
        n = _ints(rows, "rows", 4)
        self.lib.nsl_pages_read(_stream(self.index), self._p, layer, _type(k_out, rounded), _ptr(k_out), ks, _ptr(v_out), vs, _ptr(rows), n, shape[0])
        _done()

    def attn(self, layer, q, rows, out, max_rows, scale=None, window=0, work=None, rounded=False):
        """Causal attention of q [T][heads][hd] over the sequences' pages -> out (bfloat16, or float32 rounded to bf16).  Each stream and each
        captured graph has work memory of its own (40 MB); work: another one (int32).  float32 queries take part with 22 bits; rounded: they hold bf16
        values (what rope and append give with rounded=True), and 11 bits do.  NaN in a row whose query is finite: a wait on the
        device ran out, see status()."""
        _here(self.index, q, rows, out, work)
        qs, os, (T, heads, hd) = _rows(q, "q"), _rows(out, "out"), q.shape
        if out.shape != q.shape or hd != self.hd:
            raise ValueError(f"q, out: [T][heads][{self.hd}]")
        if work is not None and _ints(work, "work", 0) < self.attn_work.numel():
            raise ValueError(f"work: {self.attn_work.numel()} ints")
        n = _ints(rows, "rows", 4)
        stream = _stream(self.index)
        if work is None:
            work = self._work_of(stream)
        self.lib.nsl_pages_attn(stream, self._p, layer, _type(q, rounded), _ptr(q), qs, heads, hd ** -0.5 if scale is None else scale, window, _ptr(rows), n, max_rows, T,
                                _type(out, True), _ptr(out), os, _ptr(work))
        _done()

    def status(self):
        """0, or the code of a wait that ran out in an attention call (see nsl_pages_attn_status); reading clears it.  Synchronises the device."""
        torch.cuda.synchronize(self.device)
        with torch.cuda.device(self.device):
            code = self.lib.nsl_pages_attn_status()
        if code < 0:
            raise RuntimeError(self.lib.nsl_pages_error().decode())
        return code

    def extend(self, reqs, got=None):
        """Sequences grow: reqs int32 [n][2] = (sequence, length); got (int32 [n], optional): 1 where served."""
        _here(self.index, reqs, got)
        n = _ints(reqs, "reqs", 2)
        if got is not None and _ints(got, "got", 0) < n:
            raise ValueError("got: one value a request")
        self.lib.nsl_pages_extend(_stream(self.index), self._p, _ptr(reqs), n, _ptr(got))
        _done()

    def fork(self, forks):
        """forks int32 [n][4] = (source, destination, length, 0): the destination shares the source's first positions."""
        _here(self.index, forks)
        self.lib.nsl_pages_fork(_stream(self.index), self._p, _ptr(forks), _ints(forks, "forks", 4))
        _done()

    def trim(self, reqs):
        """Sequences are cut back: reqs int32 [n][2] = (sequence, length)."""
        _here(self.index, reqs)
        self.lib.nsl_pages_trim(_stream(self.index), self._p, _ptr(reqs), _ints(reqs, "reqs", 2))
        _done()

    def compact(self):
        """The pages in use move to the lowest ids; used() says how many there are."""
        _here(self.index)
        self.lib.nsl_pages_compact(_stream(self.index), self._p)
        _done()

    def used(self):
        """Pages in use (waits for the device)."""
        return int((self.ref > 0).sum())

    def copy(self, pairs):
        """Pages pairs[i][0] -> pairs[i][1] (int32 [n][2]), in all layers."""
        _here(self.index, pairs)
        self.lib.nsl_pages_copy(_stream(self.index), self._p, _ptr(pairs), _ints(pairs, "pairs", 2))
        _done()
