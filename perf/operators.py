"""The paged 8-bit KV cache and the operators around it, as cases that can be timed and compared: rotary positions, the store into
pages and the read back, attention over pages, and the pages' management.  listed() names the cases that are looked at first;
draw() gives more of the same ranges.

A pool holds, for every layer, `n_pages` pages of `page` positions: int8 codes [n_layer][n_pages][n_kv][page][hd] of keys and of
values and one float32 scale per page and head; a value is code * scale.  A sequence's row of the page table names its pages;
`ref` counts the sequences that a page belongs to, `length` the positions of a sequence.  A call's rows are given as
descriptors (first row, number of rows, position of the first, sequence).

Kinds of case:
  rope     rotary positions on the queries and keys of T rows (half or interleaved pairs, all or part of the head)
  append   rotary positions on the queries and keys, the keys and values into the pages of their sequences; then the pages that
           were written are read back as the values they hold
  attn     causal attention of each sequence's rows over its pages
  fork     sequences forked (pages shared), and the forks extended: a shared last page is copied, new pages are allotted
  compact  a pool with holes: the pages in use move to the lowest ids

In the plain form everything is computed from elementary operations in 32 bits, angles in 64."""
import math
import random

import torch

own = False

EL = {"bf16": 2, "f32": 4}
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a decode batch's queries and keys, rotated in the engine's f32 arrays: latency
        {"name": "rope_32_f32", "kind": "rope", "T": 32, "heads": 16, "kv": 2, "hd": 128, "rot": 128, "inter": False, "type": "f32", "far": 4096, "factor": 1.0},
        # a prompt of odd length far into a long context, part of the head in interleaved pairs
        {"name": "rope_5003_inter64", "kind": "rope", "T": 5003, "heads": 32, "kv": 8, "hd": 128, "rot": 64, "inter": True, "type": "bf16", "far": 900000, "factor": 1.14},
        # one token of each of 32 sequences into its last page
        {"name": "append_32x1", "kind": "append", "S": 32, "rows": 1, "even": True, "ctx": 4096, "heads": 16, "kv": 2, "hd": 128, "page": 64, "rot": 128, "inter": False, "type": "f32"},
        # chunks of prompts of different lengths
        {"name": "append_6_ragged700", "kind": "append", "S": 6, "rows": 700, "even": False, "ctx": 2000, "heads": 32, "kv": 4, "hd": 64, "page": 16, "rot": 32, "inter": True, "type": "bf16"},
        # a long prompt in one call
        {"name": "append_1x8192", "kind": "append", "S": 1, "rows": 8192, "even": True, "ctx": 0, "heads": 16, "kv": 8, "hd": 128, "page": 64, "rot": 128, "inter": False, "type": "bf16"},
        # single-stream decode: the smallest call
        {"name": "attn_1x1_900", "kind": "attn", "S": 1, "rows": 1, "even": True, "ctx": 900, "heads": 16, "kv": 2, "hd": 128, "page": 64, "window": 0, "type": "f32"},
        # a decode batch of 32 sequences of different lengths (the heads and the batch of the benchmark's decoder)
        {"name": "attn_32x1_4096", "kind": "attn", "S": 32, "rows": 1, "even": True, "ctx": 4096, "heads": 16, "kv": 2, "hd": 128, "page": 64, "window": 0, "type": "f32"},
        # long contexts over small pages
        {"name": "attn_8x1_16001_page16", "kind": "attn", "S": 8, "rows": 1, "even": True, "ctx": 16001, "heads": 32, "kv": 8, "hd": 128, "page": 16, "window": 0, "type": "bf16"},
        # a step that verifies up to six drafted tokens of each sequence, narrow heads
        {"name": "attn_16x6_5000_hd64", "kind": "attn", "S": 16, "rows": 6, "even": False, "ctx": 5000, "heads": 32, "kv": 4, "hd": 64, "page": 32, "window": 0, "type": "bf16"},
        # a chunk of a long prompt behind as many positions
        {"name": "attn_1x4096_4096", "kind": "attn", "S": 1, "rows": 4096, "even": True, "ctx": 4096, "heads": 16, "kv": 2, "hd": 128, "page": 64, "window": 0, "type": "bf16"},
        # 8 sequences forked four ways each, every fork given room for its next tokens, over eight layers
        {"name": "fork_8x4", "kind": "fork", "S": 8, "width": 4, "ctx": 1000, "grow": 70, "layers": 8, "kv": 2, "hd": 128, "page": 64},
        # a pool of eight layers that is a third empty
        {"name": "compact_24x20", "kind": "compact", "S": 24, "P": 20, "live": 0.66, "layers": 8, "kv": 2, "hd": 128, "page": 64},
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], its logarithm uniform."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attn", "attn", "attn", "attn", "fork", "compact"])
    heads, kv = rng.choice([(16, 2), (32, 8), (32, 4), (8, 8), (12, 4), (24, 2), (16, 1), (40, 8)])
    hd, page, typ = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128]), rng.choice(["bf16", "f32"])
    if kind == "rope":
        return {"kind": kind, "T": _log(rng, 1, 5003), "heads": heads, "kv": kv, "hd": hd, "rot": rng.choice([hd, hd // 2, hd // 4]), "inter": rng.random() < 0.5, "type": typ,
                "far": _log(rng, 1000, 1000000), "factor": rng.choice([1.0, 1.0, 1.2])}
    if kind == "append":
        rows = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 4000)])
        return {"kind": kind, "S": _log(rng, 1, 64 if rows < 9 else max(1, 8000 // rows)), "rows": rows, "even": rng.random() < 0.5, "ctx": rng.choice([0, _log(rng, 1, 5000)]), "heads": heads,
                "kv": kv, "hd": hd, "page": page, "rot": rng.choice([hd, hd // 2]), "inter": rng.random() < 0.5, "type": typ}
    if kind == "attn":
        rows = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 3000)])
        S = _log(rng, 1, 64) if rows == 1 else _log(rng, 1, 16) if rows < 9 else rng.randint(1, 3)
        most = min(32000, 800000 // (S * kv), int(4.0e8 / (S * rows * heads)))
        return {"kind": kind, "S": S, "rows": rows, "even": rng.random() < 0.5, "ctx": rng.choice([0, 1, 1, 1]) * _log(rng, 1, max(64, most)), "heads": heads, "kv": kv, "hd": hd, "page": page,
                "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]), "type": typ}
    if kind == "fork":
        return {"kind": kind, "S": rng.randint(1, 12), "width": rng.randint(1, 6), "ctx": _log(rng, 20, 1500), "grow": rng.randint(1, 100), "layers": rng.randint(1, 8), "kv": rng.choice([1, 2, 4]),
                "hd": hd, "page": page}
    return {"kind": kind, "S": 2 * rng.randint(1, 20), "P": rng.randint(1, 20), "live": rng.uniform(0.2, 0.9), "layers": rng.randint(1, 8), "kv": rng.choice([1, 2]), "hd": hd, "page": page}


def _seqs(c):
    """(rows, position of the first) of a case's sequences: a matter of the case, not of the seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    got = []
    for _ in range(c["S"]):
        n = c["rows"] if c["even"] else rng.randint(1, c["rows"])
        got.append((n, c["ctx"] if c["S"] == 1 else rng.randint(c["ctx"] // 2, c["ctx"])))
    return got


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _up(a, b):
    return -(-a // b)


class _State:
    pass


def _pool(st, gen, layers, n_pages, kv, hd, page):
    """Codes and scales as a used cache holds them."""
    shape = (layers, n_pages, kv, page, hd)
    make = lambda: (torch.randn(shape, generator=gen, device="cuda") * 36).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    st.kc, st.vc = make(), make()
    scale = lambda: torch.exp2(torch.randint(-6, -3, shape[:3], generator=gen, device="cuda").float())  # noqa: E731
    st.ks, st.vs = scale(), scale()


def _inv(rot):
    return torch.tensor([1e6 ** (-2.0 * p / rot) for p in range(rot // 2)], dtype=torch.float64).float().cuda()


def prepare(case, seed):
    c, kind, st = case, case["kind"], _State()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16).to(DT[c["type"]])  # noqa: E731
    st.case = c
    hd, kv = c["hd"], c["kv"]
    if kind == "rope":
        T = c["T"]
        st.q, st.k, st.inv = rnd(T, c["heads"], hd), rnd(T, kv, hd), _inv(c["rot"])
        first = int(torch.randint(0, c["far"], (1,), generator=gen, device="cuda"))
        st.pos = torch.randint(0, c["far"], (T,), generator=gen, device="cuda", dtype=torch.int32) if T <= 64 else torch.arange(first, first + T, device="cuda", dtype=torch.int32)
        st.qo, st.ko = torch.empty_like(st.q), torch.empty_like(st.k)
    elif kind in ("append", "attn"):
        page, seqs = c["page"], _seqs(c)
        st.T = sum(n for n, _ in seqs)
        st.most = max(n for n, _ in seqs)
        pages = [_up(p + n, page) for n, p in seqs]
        n_pages = sum(pages) + 5
        _pool(st, gen, 2, n_pages, kv, hd, page)
        ids = torch.randperm(n_pages, generator=gen, device="cuda").int()
        st.table = torch.full((c["S"], max(pages) + 1), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(pages):
            st.table[i, :n] = ids[at:at + n]
            at += n
        st.ref = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        st.ref[ids[:at].long()] = 1
        st.length = _int([n + p for n, p in seqs])
        row, desc, back, at = 0, [], [], 0
        for i, (n, p) in enumerate(seqs):
            desc.append([row, n, p, i])
            lo = p // page * page
            back.append([at, p + n - lo, lo, i])
            row, at = row + n, at + p + n - lo
        st.rows, st.back, st.n_back, st.most_back = _int(desc), _int(back), at, max(b[1] for b in back)
        st.q = rnd(st.T, c["heads"], hd)
        if kind == "append":
            st.k, st.v, st.inv, st.qo = rnd(st.T, kv, hd), rnd(st.T, kv, hd), _inv(c["rot"]), torch.empty_like(st.q)
            st.kb, st.vb = (torch.empty((st.n_back, kv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        else:
            st.o = torch.empty(st.q.shape, dtype=torch.bfloat16, device="cuda")
    elif kind == "fork":
        page, S, W = c["page"], c["S"], c["width"]
        n = _up(c["ctx"], page)
        n_pages = S * n + S * W * (_up(c["grow"], page) + 2) + 3
        _pool(st, gen, c["layers"], n_pages, kv, hd, page)
        ids = torch.randperm(n_pages, generator=gen, device="cuda").int()
        st.table = torch.full((S * (1 + W), _up(c["ctx"] + c["grow"], page)), -1, dtype=torch.int32, device="cuda")
        st.table[:S, :n] = ids[:S * n].view(S, n)
        st.ref = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        st.ref[ids[:S * n].long()] = 1
        st.length = torch.zeros(S * (1 + W), dtype=torch.int32, device="cuda")
        st.length[:S] = c["ctx"]
        cut = torch.randint(max(1, c["ctx"] // 2), c["ctx"] + 1, (S * W,), generator=gen, device="cuda").int()
        dst = torch.arange(S, S * (1 + W), device="cuda").int()
        zero = torch.zeros_like(dst)
        st.drops, st.forks, st.grows = torch.stack([dst, zero], 1), torch.stack([(dst - S) % S, dst, cut, zero], 1), torch.stack([dst, cut + c["grow"]], 1)
        st.got = torch.zeros(S * W, dtype=torch.int32, device="cuda")
    else:
        S, P, page, half = c["S"], c["P"], c["page"], c["P"] // 2      # sequences 2 i and 2 i + 1 share their first half
        used = S // 2 * half + S * (P - half)
        n_pages = max(used, round(used / c["live"]))
        _pool(st, gen, c["layers"], n_pages, kv, hd, page)
        ids = torch.randperm(n_pages, generator=gen, device="cuda").int()[:used]
        shared = ids[:S // 2 * half].view(S // 2, half).repeat_interleave(2, 0)
        st.table0 = torch.cat([shared, ids[S // 2 * half:].view(S, P - half), torch.full((S, 2), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
        st.ref0 = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        st.ref0[ids.long()] = 1
        st.ref0[ids[:S // 2 * half].long()] = 2
        st.table, st.ref = st.table0.clone(), st.ref0.clone()
        st.length = torch.full((S,), P * page, dtype=torch.int32, device="cuda") - torch.randint(0, page, (S,), generator=gen, device="cuda").int()
    if own:
        from nanoseedlm_b200 import pages
        st.pages = pages
        if kind in ("rope", "append"):
            st.rope = pages.Rope(st.inv, interleaved=c["inter"], factor=c.get("factor", 1.0))
        if kind != "rope":
            st.pool = pages.PagePool(st.kc, st.vc, st.ks, st.vs, st.ref, st.table, st.length)
    torch.cuda.synchronize()
    return st


# ---- the plain form ---------------------------------------------------------------------------------------------------------
def _rotate(x, pos, inv, inter, factor):
    """x [T][heads][hd] in 32 bits, the angles in 64."""
    rot = 2 * inv.numel()
    a = pos.double()[:, None] * inv.double()
    cs, sn = (a.cos() * factor).float()[:, None], (a.sin() * factor).float()[:, None]
    x = x.float()
    u, w = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, r = u * cs - w * sn, w * cs + u * sn
    turned = torch.stack([p, r], -1).flatten(-2) if inter else torch.cat([p, r], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _row_of(st):
    """Of each of a call's rows: its sequence's descriptor, and its position."""
    d = torch.searchsorted(st.rows[:, 0].contiguous(), torch.arange(st.T, device="cuda", dtype=torch.int32), right=True) - 1
    return d, st.rows[d, 2] + torch.arange(st.T, device="cuda") - st.rows[d, 0]


def _plain_append(st):
    c, page, kv = st.case, st.case["page"], st.case["kv"]
    d, pos = _row_of(st)
    q = _rotate(st.q, pos, st.inv, c["inter"], 1.0).to(DT[c["type"]])
    new = [_rotate(st.k, pos, st.inv, c["inter"], 1.0), st.v.float()]
    pid = st.table[st.rows[d, 3], pos // page].long()
    # the pages that the call writes, per sequence; a page starts afresh where the call writes its first position
    lo, hi = st.rows[:, 2] // page, (st.rows[:, 2] + st.rows[:, 1] - 1) // page
    j = torch.minimum(lo[:, None] + torch.arange(_up(st.most, page) + 1, device="cuda"), hi[:, None])
    touched = torch.gather(st.table[st.rows[:, 3]], 1, j.long()).long()
    fresh = j * page >= st.rows[:, 2, None]
    for x, codes, scales in zip(new, (st.kc[1], st.vc[1]), (st.ks[1], st.vs[1])):
        top = torch.zeros_like(scales).scatter_reduce(0, pid[:, None].expand(-1, kv), x.abs().amax(-1), "amax")[touched]
        m, e = torch.frexp(top)
        e = torch.where(m <= 127 / 128, e - 7, e - 6).clamp(-126, 127)
        need = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), torch.full_like(top, 2.0 ** -126))
        old = torch.where(fresh[..., None], torch.zeros_like(top), scales[touched])
        scale = torch.maximum(need, old)
        kept = torch.round(codes[touched].float() * (old / scale)[..., None, None]).to(torch.int8)
        codes[touched] = kept
        scales[touched] = scale
        codes[pid, :, pos % page] = torch.round(x / scales[pid][..., None]).clamp(-127, 127).to(torch.int8)
    at = torch.searchsorted(st.back[:, 0].contiguous(), torch.arange(st.n_back, device="cuda", dtype=torch.int32), right=True) - 1
    pos = st.back[at, 2] + torch.arange(st.n_back, device="cuda") - st.back[at, 0]
    pid = st.table[st.back[at, 3], pos // page].long()
    k, v = ((codes[pid, :, pos % page].float() * scales[pid][..., None]).to(torch.bfloat16) for codes, scales in ((st.kc[1], st.ks[1]), (st.vc[1], st.vs[1])))
    return {"q": q, "k": k, "v": v}


def _plain_attn(st):
    c, page, kv, hd = st.case, st.case["page"], st.case["kv"], st.case["hd"]
    d, _ = _row_of(st)
    ids = st.table[st.rows[:, 3]].clamp(min=0).long()
    deq = lambda codes, scales: (codes[ids].float() * scales[ids][..., None, None]).permute(0, 2, 1, 3, 4).flatten(2, 3)  # noqa: E731
    k, v = deq(st.kc[1], st.ks[1]), deq(st.vc[1], st.vs[1])      # [S][kv][keys][hd]
    i = torch.arange(st.most, device="cuda")
    q = st.q.float()[(st.rows[:, 0, None] + i).clamp(max=st.T - 1)]      # [S][rows][heads][hd]
    S, R, H = q.shape[:3]
    q = q.view(S, R, kv, H // kv, hd).permute(0, 2, 1, 3, 4).reshape(S, kv, R * (H // kv), hd)
    s = (q @ k.transpose(-1, -2)).view(S, kv, R, H // kv, -1) * (1 / math.sqrt(hd))
    key, pos = torch.arange(k.shape[2], device="cuda"), (st.rows[:, 2, None] + i)[:, None, :, None, None]
    seen = key <= pos
    if c["window"]:
        seen &= key > pos - c["window"]
    s = s.masked_fill(~seen, -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(S, kv, R * (H // kv), -1) @ v).view(S, kv, R, H // kv, hd).permute(0, 2, 1, 3, 4).reshape(S, R, H, hd)
    return o[d, torch.arange(st.T, device="cuda") - st.rows[d, 0]].to(torch.bfloat16)


def _plain_fork(st):
    c, page = st.case, st.case["page"]
    width = st.table.shape[1]
    j = torch.arange(width, device="cuda")
    n_pages = st.ref.numel()

    def count(ids, on, by):      # ref of the pages `ids` where `on`
        st.ref.index_add_(0, ids.clamp(min=0).flatten().long(), (on.int() * by).flatten())

    seq = st.drops[:, 0].long()
    count(st.table[seq], j < ((st.length[seq] + page - 1) // page)[:, None], -1)
    st.table[seq], st.length[seq] = -1, 0
    src, dst = st.forks[:, 0].long(), st.forks[:, 1].long()
    n = torch.minimum(st.forks[:, 2], st.length[src])
    keep = j < ((n + page - 1) // page)[:, None]
    st.table[dst] = torch.where(keep, st.table[src], -1)
    count(st.table[src], keep, 1)
    st.length[dst] = n
    seq, new = st.grows[:, 0].long(), st.grows[:, 1]
    old, mine = st.length[seq], st.table[seq]
    new = torch.maximum(new, old)
    have, need, last = (old + page - 1) // page, (new + page - 1) // page, old // page
    fits = need <= width
    page_of = torch.gather(mine, 1, last.clamp(max=width - 1)[:, None].long())[:, 0].long()
    part = (old % page != 0) & (new > old) & fits
    same = (page_of[:, None] == page_of) & part & part[:, None]
    copy = part & (st.ref[page_of.clamp(min=0)] - same.tril(-1).sum(1) > 1)      # the last of those who share it keeps it
    want = torch.where(fits, need - have + copy.int(), 0)
    before = want.cumsum(0) - want
    free = torch.where(st.ref == 0, torch.arange(n_pages, device="cuda"), n_pages).sort().values
    ok = (before + want <= (st.ref == 0).sum()) & fits
    pick = before[:, None] + torch.where(j == last[:, None], 0, copy.int()[:, None] + j - have[:, None])
    fresh = ((j >= have[:, None]) & (j < need[:, None]) | (j == last[:, None]) & copy[:, None]) & ok[:, None]
    table = torch.where(fresh, free[pick.clamp(0, n_pages - 1)].int(), mine)
    st.table[seq] = table
    count(page_of, copy & ok, -1)
    count(table, fresh, 1)
    st.length[seq] = torch.where(ok, new, old)
    kept = st.table[0, 0].long()      # a page in use, for requests that copy nothing
    to = torch.where(copy & ok, torch.gather(table, 1, last.clamp(max=width - 1)[:, None].long())[:, 0].long(), kept)
    at = torch.where(copy & ok, page_of, kept)
    for x in (st.kc, st.vc, st.ks, st.vs):
        x[:, to] = x[:, at]
    st.got.copy_(ok)
    return [st.table, st.ref, st.length, st.got, st.kc, st.vc, st.ks, st.vs]


def _plain_compact(st):
    n = st.ref0.numel()
    ids = torch.arange(n, device="cuda")
    live = st.ref0 > 0
    used = live.sum()
    free = torch.where(live, n, ids).sort().values
    rank = live.long().cumsum(0) - 1
    below = (live & (ids < used)).sum()
    to = torch.where(live & (ids >= used), free[(rank - below).clamp(0, n - 1)].clamp(max=n - 1), ids)
    at = torch.cat([ids, ids[:1]]).scatter(0, torch.where(live, to, n), ids)[:n]      # what each page holds afterwards
    at = torch.where(ids < used, at, ids)
    ref = torch.where(ids < used, st.ref0[at], 0)
    table = torch.where(st.table0 >= 0, to[st.table0.clamp(min=0).long()].int(), -1)
    return [table, ref, st.length] + [x[:, at] for x in (st.kc, st.vc, st.ks, st.vs)]


def run(st):
    c, kind = st.case, st.case["kind"]
    if kind == "rope":
        if own:
            st.pages.rope(st.rope, st.q, st.k, st.pos, st.qo, st.ko)
            return {"q": st.qo, "k": st.ko}
        return {n: _rotate(x, st.pos, st.inv, c["inter"], c["factor"]).to(x.dtype) for n, x in (("q", st.q), ("k", st.k))}
    if kind == "append":
        if own:
            st.pool.append(1, st.rope, st.q, st.k, st.v, st.rows, st.qo)
            st.pool.read(1, st.back, st.kb, st.vb)
            return {"q": st.qo, "k": st.kb, "v": st.vb}
        return _plain_append(st)
    if kind == "attn":
        if own:
            st.pool.attn(1, st.q, st.rows, st.o, max_rows=st.most, window=c["window"])
            return st.o
        return _plain_attn(st)
    if kind == "fork":
        if own:
            st.pool.trim(st.drops)
            st.pool.fork(st.forks)
            st.pool.extend(st.grows, st.got)
            return [st.table, st.ref, st.length, st.got, st.kc, st.vc, st.ks, st.vs]
        return _plain_fork(st)
    if own:
        st.table.copy_(st.table0)
        st.ref.copy_(st.ref0)
        st.pool.compact()
        return [st.table, st.ref, st.length, st.kc, st.vc, st.ks, st.vs]
    return _plain_compact(st)


def work(case):
    c, kind, hd, kv = case, case["kind"], case["hd"], case["kv"]
    if kind == "rope":
        n = c["T"] * (c["heads"] + kv)
        return {"bytes": 2 * n * hd * EL[c["type"]] + 4 * c["T"] + 2 * c["rot"], "flops": 3.0 * n * c["rot"]}
    page = c["page"]
    if kind == "append":
        T = sum(n for n, _ in _seqs(c))
        back = sum(n + p % page for n, p in _seqs(c))
        row, el = kv * hd, EL[c["type"]]
        return {"bytes": T * (2 * c["heads"] * hd * el + 2 * row * el + 2 * row) + back * row * 2 * (1 + 2), "flops": 3.0 * T * (c["heads"] + kv) * c["rot"] + 4.0 * T * row}
    if kind == "attn":
        nbytes = flops = 0
        for n, p in _seqs(c):
            w = c["window"] or p + n
            seen = sum(min(p + i + 1, w) for i in range(n))
            keys = min(p + n, w + n - 1)
            nbytes += keys * kv * 2 * hd + 8 * kv * (keys // page + 1) + n * c["heads"] * hd * (EL[c["type"]] + 2)
            flops += 4.0 * hd * c["heads"] * seen
        return {"bytes": nbytes, "flops": flops}
    one = 2 * c["layers"] * kv * (page * hd + 4)      # a page's codes and scales in all layers
    if kind == "fork":
        n = c["S"] * c["width"]
        return {"bytes": 2 * n * one + 4 * 2 * n * (_up(c["ctx"], page) + _up(c["grow"], page)), "flops": 0}
    half = c["P"] // 2
    used = c["S"] // 2 * half + c["S"] * (c["P"] - half)
    total = max(used, round(used / c["live"]))
    return {"bytes": 2 * one * used * (1 - used / total) + 8 * total + 8 * c["S"] * c["P"], "flops": 0}


# ---- the definition, in 64 bits ---------------------------------------------------------------------------------------------
def _turn64(x, pos, inv, inter, factor):
    x = x.double().clone()
    rot = 2 * inv.numel()
    z = torch.polar(torch.full((pos.numel(), inv.numel()), float(factor), dtype=torch.float64, device="cuda"), pos.double()[:, None] * inv.double())[:, None]
    at = torch.arange(inv.numel(), device="cuda")
    a, b = (2 * at, 2 * at + 1) if inter else (at, at + rot // 2)
    y = torch.complex(x[..., a], x[..., b]) * z
    x[..., a], x[..., b] = y.real, y.imag
    return x


def exact(case, seed):
    c, kind = case, case["kind"]
    if kind in ("fork", "compact"):
        return None      # whole numbers and copies
    st = prepare(case, seed)
    if kind == "rope":
        return {"q": _turn64(st.q, st.pos, st.inv, c["inter"], c["factor"]), "k": _turn64(st.k, st.pos, st.inv, c["inter"], c["factor"])}
    page, hd, kv = c["page"], c["hd"], c["kv"]
    out, ks, vs = [], [], []
    for row, n, p, s in st.rows.tolist():
        pos = torch.arange(p, p + n, device="cuda")
        if kind == "append":
            sides = []
            out.append(_turn64(st.q[row:row + n], pos, st.inv, c["inter"], 1.0))
            for x, codes, scales in ((_turn64(st.k[row:row + n], pos, st.inv, c["inter"], 1.0), st.kc[1], st.ks[1]), (st.v[row:row + n].double(), st.vc[1], st.vs[1])):
                held = []
                for j in range(p // page, (p + n - 1) // page + 1):
                    lo, hi = max(p, j * page), min(p + n, (j + 1) * page)
                    mine, old = x[lo - p:hi - p], scales[st.table[s, j]].double()
                    need = torch.exp2(torch.ceil(torch.log2(mine.abs().amax((0, 2)) / 127)))
                    scale = need if lo == j * page else torch.maximum(need, old)
                    if lo > j * page:
                        was = codes[st.table[s, j], :, :lo - j * page].double()
                        held.append((torch.round(was * (old / scale)[:, None, None]) * scale[:, None, None]).transpose(0, 1))
                    held.append(torch.round(mine / scale[:, None]) * scale[:, None])
                sides.append(torch.cat(held))
            ks.append(sides[0])
            vs.append(sides[1])
            continue
        ids = st.table[s, :_up(p + n, page)].long()
        k, v = ((codes[1, ids].double() * scales[1, ids].double()[..., None, None]).transpose(0, 1).reshape(kv, -1, hd) for codes, scales in ((st.kc, st.ks), (st.vc, st.vs)))
        heads = []
        for h in range(c["heads"]):
            g = h // (c["heads"] // kv)
            x = st.q[row:row + n, h].double() @ k[g].T / math.sqrt(hd)
            key = torch.arange(k.shape[1], device="cuda")
            off = key[None] > pos[:, None]
            if c["window"]:
                off |= key[None] <= pos[:, None] - c["window"]
            heads.append(torch.softmax(x.masked_fill(off, -math.inf), -1) @ v[g])
        out.append(torch.stack(heads, 1))
    if kind == "attn":
        return torch.cat(out)
    return {"q": torch.cat(out), "k": torch.cat(ks), "v": torch.cat(vs)}
