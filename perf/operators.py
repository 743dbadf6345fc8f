"""The 4-bit paged KV cache operators as they are measured: their cases, their plain
forms in elementary torch operations, and the calls a user makes of them.

The cache.  A page holds `page` tokens (a multiple of 16) of every kv head.  Per kv head
a page is a run of 1152-byte cells, [page / 16][head_dim / 64]: one cell is 16 tokens x
64 dims of K and of V.

  bytes    0..511   K codes   [t % 8][c][t / 8][8 bytes], dim = 16 c + 2 byte + nibble
  bytes  512..1023  V codes   [g][c][p][quad][e][2 bytes], token = 8 p + 2 c + e,
                              dim = 8 g + 4 quad + 2 byte + nibble
  bytes 1024..1087  K d and m [t % 8][t / 8] pairs of bf16
  bytes 1088..1151  V d and m, the same

A value is code * d + m; every (token, kv head, 64 dims) has its own d and m:
  m = bf16(min x), d = max(bf16((max x - m) / 15), 2^-40),
  code = clamp(floor((x - m) / d + 1/2), 0, 15).

Operators: append (rotation, quantisation, page summaries) with gather (the values read
back), decode (attention of one query per sequence), select + decode (the same over the
pages that a bound on their scores picks), reorder (fork, free and reserve pages of the
rows of a page table) and compact (live pages to the lowest ids)."""

import math

import torch

own = False

CELL = 1152
D_MIN = 2.0 ** -40

# Head layouts: (q heads, kv heads, head_dim) of the dense 3B decoder and of the gated
# full-attention layers, and two generic ones (head_dim 128; as many kv heads as q heads).
LAYOUTS = [(40, 8, 64), (8, 2, 256), (32, 8, 128), (8, 8, 64)]


def listed():
    return [
        # chat with one user: the shortest decode call, all latency
        dict(name="decode b1 c512", op="decode", batch=1, hq=40, hkv=8, dim=64, ctx=512, page=64, ragged=False),
        # a server's mixed batch: lengths from 1 to 4096 and small pages
        dict(name="decode b16 ragged", op="decode", batch=16, hq=40, hkv=8, dim=64, ctx=4096, page=16, ragged=True),
        # the dense decoder's large batch at its context
        dict(name="decode b64 c4096", op="decode", batch=64, hq=40, hkv=8, dim=64, ctx=4096, page=64, ragged=False),
        # the hybrid stack's attention layers at their large decode batch
        dict(name="decode b256 d256", op="decode", batch=256, hq=8, hkv=2, dim=256, ctx=2048, page=64, ragged=False),
        # one long conversation, 2048 of its 32768 tokens attended
        dict(name="sparse b1 c32768", op="sparse", batch=1, hq=40, hkv=8, dim=64, ctx=32768, page=64, n_sel=32,
             ragged=False),
        # long documents in a batch, lengths mixed
        dict(name="sparse b16 ragged", op="sparse", batch=16, hq=40, hkv=8, dim=64, ctx=32768, page=32, n_sel=64,
             ragged=True),
        # the new token of every sequence of a decode step
        dict(name="append step b64", op="append", batch=64, hkv=8, dim=64, page=64, rows=64, dtype="float32",
             rope=True),
        # prompts of four users arriving together, at odd lengths, behind what they have
        dict(name="append prompts 8192", op="append", batch=4, hkv=8, dim=64, page=64, rows=8192, dtype="float32",
             rope=True),
        # a beam step of one request
        dict(name="reorder b8", op="reorder", batch=8, layers=40, hkv=8, dim=64, page=16, ctx=512),
        # a beam step of a full server
        dict(name="reorder b64", op="reorder", batch=64, layers=8, hkv=8, dim=64, page=64, ctx=2048),
        # a small pool after a few requests ended
        dict(name="compact 256", op="compact", batch=8, layers=8, hkv=2, dim=256, page=16, pages=256),
        # a server's pool, 40% freed
        dict(name="compact 2048", op="compact", batch=48, layers=6, hkv=8, dim=64, page=64, pages=2048),
    ]


def _spread(rng, lo, hi):
    """An integer in lo..hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "sparse", "append", "reorder", "compact"])
    hq, hkv, dim = rng.choice(LAYOUTS)
    page = rng.choice([16, 32, 64, 128])
    if op in ("decode", "sparse"):
        ctx = _spread(rng, 1, 32768) if op == "decode" else _spread(rng, 64, 32768)
        most = min(256, max(1, 268435456 // (ctx * hkv * dim)))
        case = dict(op=op, batch=_spread(rng, 1, most), hq=hq, hkv=hkv, dim=dim, ctx=ctx, page=page,
                    ragged=rng.random() < 0.5)
        if op == "sparse":
            case["n_sel"] = rng.randint(1, min(96, 2048 // page))
        return case
    if op == "append":
        batch = _spread(rng, 1, 64)
        rows = batch if rng.random() < 0.3 else max(batch, _spread(rng, 1, 4194304 // (hkv * dim)))
        return dict(op=op, batch=batch, hkv=hkv, dim=dim, page=page, rows=rows,
                    dtype=rng.choice(["float32", "bfloat16"]), rope=rng.random() < 0.7)
    if op == "reorder":
        return dict(op=op, batch=_spread(rng, 1, 64), layers=rng.randint(1, 8), hkv=hkv, dim=dim, page=page,
                    ctx=_spread(rng, 16, 1048576 // (hkv * dim)))
    return dict(op=op, batch=_spread(rng, 1, 64), layers=rng.randint(1, 6), hkv=hkv, dim=dim, page=page,
                pages=_spread(rng, 16, 2097152 // (hkv * dim * page // 64 * 2)))


# ---------------------------------------------------------------- inputs

def _quantise(x):
    """x [..., 64] -> codes uint8 and (d, m) bf16 [..., 2], in the type x has."""
    m = x.amin(-1, keepdim=True).float().bfloat16()
    d = ((x.amax(-1, keepdim=True) - m.to(x.dtype)) / 15).float().bfloat16().clamp(min=D_MIN)
    code = ((x - m.to(x.dtype)) / d.to(x.dtype) + 0.5).floor().clamp(0, 15).to(torch.uint8)
    return code, torch.cat([d, m], -1)


def _cells(kc, km, vc, vm):
    """Codes [..., 16, 64] and (d, m) [..., 16, 2] of K and V -> cells [..., 1152]."""
    lead = kc.shape[:-2]
    n = len(lead)
    at = list(range(n))
    k = kc.reshape(*lead, 2, 8, 4, 8, 2)
    k = (k[..., 0] | (k[..., 1] << 4)).permute(*at, n + 1, n + 2, n, n + 3).reshape(*lead, 512)
    v = vc.reshape(*lead, 2, 4, 2, 8, 2, 2, 2)
    v = (v[..., 0] | (v[..., 1] << 4)).permute(*at, n + 3, n + 1, n, n + 4, n + 2, n + 5).reshape(*lead, 512)
    meta = [x.reshape(*lead, 2, 8, 2).transpose(n, n + 1).contiguous().view(torch.uint8).reshape(*lead, 64)
            for x in (km, vm)]
    return torch.cat([k, v, *meta], -1)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _total(case):
    """Lengths in 1..ctx: evenly spread where they are ragged, else a few tokens short of ctx at most."""
    b, ctx = case["batch"], case["ctx"]
    if case["ragged"]:
        return [1 + int((ctx - 1) * (i + 0.5) / b) for i in range(b)]
    return [max(1, ctx - i % 7) for i in range(b)]


def _lengths(case, g):
    n = torch.tensor(_total(case), device="cuda", dtype=torch.int32)
    return n[torch.randperm(n.numel(), device="cuda", generator=g)]


def _tables(lens, page, n_pages, most, g):
    """A page table [B, most] over pages placed at random among n_pages, -1 behind a row's pages."""
    need = (lens.long() + page - 1) // page
    used = torch.arange(most, device="cuda") < need[:, None]
    table = torch.full((lens.numel(), most), -1, dtype=torch.int32, device="cuda")
    table[used] = torch.randperm(n_pages, device="cuda", generator=g)[:int(need.sum())].to(torch.int32)
    return table


def _filled(n_pages, hkv, dim, page, g):
    """A pool of pages with quantised keys and values, and the pages' key summaries.  Keys have
    channels of unlike size, as rotated keys do; values are near normal."""
    cell = (n_pages, hkv, page // 16, 16, dim)
    size = torch.exp(0.5 * torch.randn(hkv, 1, 1, dim, device="cuda", generator=g))
    k = torch.randn(cell, device="cuda", generator=g) * size
    summary = torch.stack([k.amin((2, 3)), k.amax((2, 3))], 2).bfloat16()
    k = k.reshape(*cell[:-1], dim // 64, 64).transpose(3, 4)
    kc, km = _quantise(k)
    del k
    v = torch.randn(*cell[:3], dim // 64, 16, 64, device="cuda", generator=g)
    vc, vm = _quantise(v)
    del v
    return _cells(kc, km, vc, vm).reshape(n_pages, hkv, -1), summary


def prepare(case, seed):
    g = _generator(seed)
    return {"decode": _prepare_decode, "sparse": _prepare_decode, "append": _prepare_append,
            "reorder": _prepare_reorder, "compact": _prepare_compact}[case["op"]](case, g)


def _prepare_decode(case, g):
    lens = _lengths(case, g)
    pages = [-(-n // case["page"]) for n in _total(case)]
    n_pages = sum(pages) + 3
    table = _tables(lens, case["page"], n_pages, max(pages), g)
    pool, summary = _filled(n_pages, case["hkv"], case["dim"], case["page"], g)
    # q is a slice of the projection's rows, as the decoder has it
    qkv = torch.randn(case["batch"], (case["hq"] + 2 * case["hkv"]) * case["dim"], device="cuda", generator=g)
    return dict(case=case, q=qkv[:, :case["hq"] * case["dim"]], pool=pool, summary=summary, table=table,
                pos=lens - 1)


def _prepare_append(case, g):
    b, hkv, dim, page, rows = (case[x] for x in ("batch", "hkv", "dim", "page", "rows"))
    dtype = getattr(torch, case["dtype"])
    if rows == b:
        new = torch.ones(b, dtype=torch.int32, device="cuda")
    else:  # rows split at random places, every sequence with one at least
        cuts = torch.randperm(rows - 1, device="cuda", generator=g)[:b - 1].sort().values.to(torch.int32) + 1
        edge = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), rows)])
        new = edge[1:] - edge[:-1]
    pos = torch.randint(0, 2048, (b,), device="cuda", generator=g, dtype=torch.int32)
    n_pages = -(-rows // page) + b * (2048 // page + 1)
    table = _tables(pos + new, page, n_pages, -(-(2048 + rows) // page), g)
    size = torch.exp(0.5 * torch.randn(hkv * dim, device="cuda", generator=g))
    # k and v are slices of one projection's rows
    kv = torch.randn(rows, 2 * hkv * dim, device="cuda", generator=g)
    kv[:, :hkv * dim] *= size
    kv = kv.to(dtype)
    pool, summary = _filled(n_pages, hkv, dim, page, g)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0).to(torch.int32)])
    return dict(case=case, k=kv[:, :hkv * dim], v=kv[:, hkv * dim:], pool=pool, summary=summary, table=table, pos=pos,
                cu=None if rows == b else cu, theta=10000.0 if case["rope"] else None)


def _prepare_reorder(case, g):
    """Rows in pairs: one row of each pair goes on twice, the other's pages are freed."""
    b, page, ctx = case["batch"], case["page"], case["ctx"]
    lens = torch.randint(max(1, ctx // 2), ctx + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
    lens[::5] = (lens[::5] + page - 1) // page * page  # some rows end with their page
    n_pages = b * (-(-ctx // page) + 2) + 2
    table = _tables(lens, page, n_pages, -(-ctx // page) + 2, g)
    refs = torch.bincount(table[table >= 0].long(), minlength=n_pages).to(torch.int32)
    row = torch.arange(b, device="cuda", dtype=torch.int32)
    one = torch.randint(0, 2, ((b + 1) // 2,), device="cuda", generator=g, dtype=torch.int32)
    parent = (row // 2 * 2 + one[row.long() // 2]).clamp(max=b - 1)
    rb = case["dim"] * page // 8 * 9
    pool = torch.randint(0, 256, (case["layers"], n_pages, case["hkv"], rb), device="cuda", generator=g,
                         dtype=torch.uint8)
    summary = torch.randn(case["layers"], n_pages, case["hkv"], 2, case["dim"], device="cuda", generator=g).bfloat16()
    return dict(case=case, pool=pool, summary=summary, table=table, lens=lens, refs=refs, parent=parent,
                reserve=torch.ones_like(lens))


def _prepare_compact(case, g):
    """60% of the pages are live, anywhere in the pool, some of them in two rows."""
    b, n = case["batch"], case["pages"]
    live = max(1, 6 * n // 10)
    ids = torch.randperm(n, device="cuda", generator=g)[:live].to(torch.int32)
    most = -(-live // b) + 1
    table = torch.full((b, most), -1, dtype=torch.int32, device="cuda")
    table[:, 1:] = torch.cat([ids, ids.new_full((b * (most - 1) - live,), -1)]).reshape(b, most - 1)
    table[:, 0] = ids[0]  # a page that every row shares
    refs = torch.bincount(table[table >= 0].long(), minlength=n).to(torch.int32)
    rb = case["dim"] * case["page"] // 8 * 9
    pool = torch.randint(0, 256, (case["layers"], n, case["hkv"], rb), device="cuda", generator=g, dtype=torch.uint8)
    summary = torch.randn(case["layers"], n, case["hkv"], 2, case["dim"], device="cuda", generator=g).bfloat16()
    return dict(case=case, pool=pool, summary=summary, table=table, refs=refs)


# ---------------------------------------------------------------- the plain forms

def _turned(x, pos, theta, dim):
    """x [..., heads, dim] at positions pos [...]: half-split rotation in 64 bits."""
    half = dim // 2
    i = torch.arange(half, device=x.device, dtype=torch.float64)
    angle = pos.double()[..., None] * theta ** (-2 * i / dim)
    c, s = angle.cos()[..., None, :], angle.sin()[..., None, :]
    x = x.double()
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _values(cells):
    """Cells [..., 1152] -> K and V in 32 bits, [..., 16, 64] each."""
    lead = cells.shape[:-1]
    n = len(lead)
    at = list(range(n))
    k = cells[..., :512].reshape(*lead, 8, 4, 2, 8).permute(*at, n + 2, n, n + 1, n + 3)
    v = cells[..., 512:1024].reshape(*lead, 8, 4, 2, 2, 2, 2).permute(*at, n + 2, n + 1, n + 4, n, n + 3, n + 5)
    out = []
    for code, lo in ((k, 1024), (v, 1088)):
        code = torch.stack([code & 15, code >> 4], -1).reshape(*lead, 16, 64).float()
        dm = cells[..., lo:lo + 64].contiguous().view(torch.bfloat16).reshape(*lead, 8, 2, 2)
        dm = dm.transpose(n, n + 1).reshape(*lead, 16, 2).float()
        out.append(code * dm[..., :1] + dm[..., 1:])
    return out


def _rows_of(pool, table, page, dim):
    """The pages of table [B, N] (any id where it is -1) as K and V [B, Hkv, N * page, dim]."""
    b, n = table.shape
    hkv = pool.shape[1]
    cells = pool[table.clamp(min=0).long()].reshape(b, n, hkv, page // 16, dim // 64, CELL)
    return [x.permute(0, 2, 1, 3, 5, 4, 6).reshape(b, hkv, n * page, dim) for x in _values(cells)]


def _attend(q, k, v, seen, scale):
    """q [B, Hkv, G, dim], k and v [B, Hkv, T, dim], seen [B, 1 or Hkv, T]: softmax attention, rows
    that see nothing are zero."""
    seen = seen[:, :, None]
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - top).masked_fill(~seen, 0)
    v = v.masked_fill(~seen.transpose(-1, -2), 0)
    return (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_decode(s, sel=None):
    c = s["case"]
    b, hq, hkv, dim, page = c["batch"], c["hq"], c["hkv"], c["dim"], c["page"]
    q = _turned(s["q"].reshape(b, hq, dim), s["pos"], 10000.0, dim).float().reshape(b, hkv, hq // hkv, dim)
    at = torch.arange(page, device="cuda")
    if sel is None:
        k, v = _rows_of(s["pool"], s["table"], page, dim)
        seen = (torch.arange(k.shape[2], device="cuda") <= s["pos"][:, None])[:, None]
    else:  # every kv head has pages of its own
        n = sel.shape[2]
        ids = s["table"].long().gather(1, sel.clamp(min=0).long().reshape(b, -1)).reshape(b, hkv, n).clamp(min=0)
        cells = s["pool"][ids, torch.arange(hkv, device="cuda")[:, None]]
        cells = cells.reshape(b, hkv, n, page // 16, dim // 64, CELL)
        k, v = [x.transpose(4, 5).reshape(b, hkv, n * page, dim) for x in _values(cells)]
        seen = ((sel[..., None].long() * page + at <= s["pos"][:, None, None, None]) & (sel[..., None] >= 0))
        seen = seen.reshape(b, hkv, n * page)
    return _attend(q, k, v, seen, dim ** -0.5).reshape(b, hq * dim).bfloat16()


def _plain_select(s):
    """For each kv head the n_sel pages with the largest bound on a score of its q heads: the sum over
    dims of max(q * min, q * max), the largest over the heads.  The page of the query's own position is
    always among them; ties go to the lower page.  In 64 bits: a choice turns on the last bit."""
    c = s["case"]
    b, hq, hkv, dim, page, n_sel = c["batch"], c["hq"], c["hkv"], c["dim"], c["page"], c["n_sel"]
    q = _turned(s["q"].reshape(b, hq, dim), s["pos"], 10000.0, dim).reshape(b, hkv, hq // hkv, dim)
    n = s["table"].shape[1]
    bound = s["summary"][s["table"].clamp(min=0).long()].double()  # [B, N, Hkv, 2, dim]
    lo, hi = bound[..., 0, :].transpose(1, 2), bound[..., 1, :].transpose(1, 2)
    up, down = q.clamp(min=0), q.clamp(max=0)
    score = (up @ hi.transpose(-1, -2) + down @ lo.transpose(-1, -2)).amax(2)  # [B, Hkv, N]
    last = (s["pos"].long().clamp(min=0) // page)[:, None, None]
    j = torch.arange(n, device="cuda")
    score = score.masked_fill(j == last, math.inf).masked_fill((j > last) | (s["pos"] < 0)[:, None, None], -math.inf)
    score, at = score.sort(dim=-1, descending=True, stable=True)
    at = at.masked_fill(score == -math.inf, n)[..., :n_sel].sort(-1).values
    at = torch.cat([at, at.new_full((b, hkv, max(0, n_sel - n)), n)], -1)
    return at.masked_fill(at == n, -1).to(torch.int32)


def _new_rows(s):
    """The sequence and the position of every new row."""
    rows = s["k"].shape[0]
    if s["cu"] is None:
        seq = torch.arange(rows, device="cuda")
        return seq, s["pos"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.bucketize(row, s["cu"][1:].long(), right=True)
    return seq, s["pos"].long()[seq] + row - s["cu"].long()[seq]


def _plain_append(s):
    c = s["case"]
    hkv, dim, page = c["hkv"], c["dim"], c["page"]
    rows = s["k"].shape[0]
    seq, pos = _new_rows(s)
    where = s["table"].long()[seq, pos // page]
    k, v = s["k"].reshape(rows, hkv, dim).double(), s["v"].reshape(rows, hkv, dim).double()
    if s["theta"] is not None:
        k = _turned(k, pos, s["theta"], dim)
    # the pages' summaries: a page whose first token is new starts anew
    n_pages = s["pool"].shape[0]
    kb = k.float().bfloat16().float()
    at = where[:, None, None].expand(rows, hkv, dim)
    first = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
    first[where[pos % page == 0]] = True
    old = s["summary"].float()
    old[:, :, 0].masked_fill_(first[:, None, None], math.inf)
    old[:, :, 1].masked_fill_(first[:, None, None], -math.inf)
    low = old[:, :, 0].scatter_reduce(0, at, kb, "amin")
    high = old[:, :, 1].scatter_reduce(0, at, kb, "amax")
    s["summary"].copy_(torch.stack([low, high], 2))
    # the codes, into the cells' bytes
    t = pos % 16
    cell = s["pool"].view(n_pages, hkv, page // 16, dim // 64, CELL)
    kc, km = _quantise(k.reshape(rows, hkv, dim // 64, 64))
    vc, vm = _quantise(v.reshape(rows, hkv, dim // 64, 64))
    kb = (kc[..., 0::2] | (kc[..., 1::2] << 4)).reshape(rows, hkv, dim // 64, 32)
    vb = (vc[..., 0::2] | (vc[..., 1::2] << 4)).reshape(rows, hkv, dim // 64, 32)
    i = torch.arange(32, device="cuda")
    k_at = (t % 8 * 64 + t // 8 * 8)[:, None] + i // 8 * 16 + i % 8
    v_at = 512 + (t % 8 // 2 * 16 + t // 8 * 8 + t % 2 * 2)[:, None] + i // 4 * 64 + i // 2 % 2 * 4 + i % 2
    m_at = (t % 8 * 8 + t // 8 * 4)[:, None] + torch.arange(4, device="cuda")
    at = torch.cat([k_at, v_at, 1024 + m_at, 1088 + m_at], 1)[:, None, None, :]
    byte = torch.cat([kb, vb, km.contiguous().view(torch.uint8), vm.contiguous().view(torch.uint8)], -1)
    h = torch.arange(hkv, device="cuda")[None, :, None, None]
    grp = torch.arange(dim // 64, device="cuda")[None, None, :, None]
    cell[where[:, None, None, None], h, (pos % page // 16)[:, None, None, None], grp, at] = byte
    # and read back
    cells = cell[where[:, None], torch.arange(hkv, device="cuda"), (pos % page // 16)[:, None]]
    row = torch.arange(rows, device="cuda")
    kr, vr = [x[row, :, :, t].reshape(rows, hkv * dim).bfloat16() for x in _values(cells)]
    return dict(k=kr, v=vr, summary=s["summary"])


def _plain_reorder(s):
    page = s["case"]["page"]
    table, lens, refs, parent = s["table"], s["lens"], s["refs"], s["parent"]
    b, most = table.shape
    row, j = torch.arange(b, device="cuda"), torch.arange(most, device="cuda")
    valid, par = parent >= 0, parent.clamp(min=0).long()
    n_pages = refs.numel()
    first = ~((parent[:, None] == parent[None]) & (row[None] < row[:, None])).any(1)
    length = torch.where(valid, lens[par], 0)
    full = length // page
    old = table[par]
    kept = (j < full[:, None]) | first[:, None]
    new = old.masked_fill(~kept | ~valid[:, None], -1)
    left = refs - torch.bincount(table[table >= 0].long(), minlength=n_pages)
    left = left + torch.bincount(new[new >= 0].long(), minlength=n_pages)
    want = (length + s["reserve"].clamp(min=0) + page - 1) // page
    holes = ((new < 0) & (j < want[:, None])).nonzero()
    free = (left == 0).nonzero()[:, 0]
    n = min(holes.shape[0], free.numel())
    r, e = holes[:n].unbind(1)
    new[r, e] = free[:n].to(torch.int32)
    left[free[:n]] = 1
    copied = valid & ~first & (length % page != 0)
    got = new.gather(1, full[:, None].long().clamp(max=most - 1))[:, 0]
    short = copied & (got < 0)
    length = torch.where(short, full * page, length).to(torch.int32)
    copied &= ~short
    src = old[row, full.long().clamp(max=most - 1)][copied].long()
    dst = got[copied].long()
    s["pool"][:, dst] = s["pool"][:, src]
    s["summary"][:, dst] = s["summary"][:, src]
    lost = (want.long() - most).clamp(min=0).sum() + holes.shape[0] - n
    info = torch.stack([(left == 0).sum(), copied.sum(), lost, lost * 0]).to(torch.int32)
    return dict(table=new, lens=length, refs=left.to(torch.int32), info=info, pool=s["pool"], summary=s["summary"])


def _plain_compact(s):
    table, refs = s["table"], s["refs"]
    n = refs.numel()
    alive = refs > 0
    live = int(alive.sum())
    src = alive[live:].nonzero()[:, 0] + live
    dst = (~alive[:live]).nonzero()[:, 0]
    to = torch.arange(n, device="cuda", dtype=torch.int32)
    to[src] = dst.to(torch.int32)
    s["pool"][:, dst] = s["pool"][:, src]
    s["summary"][:, dst] = s["summary"][:, src]
    new = torch.where(table >= 0, to[table.clamp(min=0).long()], -1)
    left = refs.clone()
    left[dst] = refs[src]
    left[live:] = 0
    info = torch.tensor([live, src.numel(), 0, 0], dtype=torch.int32, device="cuda")
    return dict(table=new, refs=left, info=info, pool=s["pool"], summary=s["summary"])


def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "decode":
        return _plain_decode(s)
    if c["op"] == "sparse":
        sel = _plain_select(s)
        return dict(sel=sel, out=_plain_decode(s, sel))
    return {"append": _plain_append, "reorder": _plain_reorder, "compact": _plain_compact}[c["op"]](s)


def _run_own(s, c):
    from llmnputest_b200 import ops
    if c["op"] == "reorder":
        table, lens, refs, info = ops.kv4_reorder(s["pool"], s["table"], s["lens"], s["refs"], s["parent"],
                                                  head_dim=c["dim"], reserve=s["reserve"], summary=s["summary"])
        return dict(table=table, lens=lens, refs=refs, info=info, pool=s["pool"], summary=s["summary"])
    if c["op"] == "compact":
        table, refs, info = ops.kv4_compact(s["pool"], s["table"], s["refs"], summary=s["summary"])
        return dict(table=table, refs=refs, info=info, pool=s["pool"], summary=s["summary"])
    if c["op"] == "append":
        ops.kv4_append(s["k"], s["v"], s["pool"], s["table"], s["pos"], n_kv_heads=c["hkv"], head_dim=c["dim"],
                       cu=s["cu"], theta=s["theta"], summary=s["summary"])
        k, v = ops.kv4_gather(s["pool"], s["table"], s["pos"], s["k"].shape[0], n_kv_heads=c["hkv"],
                              head_dim=c["dim"], cu=s["cu"])
        return dict(k=k, v=v, summary=s["summary"])
    heads = dict(n_q_heads=c["hq"], n_kv_heads=c["hkv"], head_dim=c["dim"], theta=10000.0)
    if c["op"] == "decode":
        return ops.kv4_decode(s["q"], s["pool"], s["table"], s["pos"], **heads)
    sel = ops.kv4_select(s["q"], s["summary"], s["table"], s["pos"], page=c["page"], n_sel=c["n_sel"], **heads)
    return dict(sel=sel, out=ops.kv4_decode(s["q"], s["pool"], s["table"], s["pos"], select=sel, **heads))


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    hkv, dim, page, b = case["hkv"], case["dim"], case["page"], case["batch"]
    row = hkv * dim * 9 // 8  # bytes of one token's K and V
    page_bytes = page * row + 4 * hkv * dim  # with its summary
    if case["op"] in ("decode", "sparse"):
        hq = case["hq"]
        lens = _total(case)
        io = b * hq * dim * (4 + 2) + sum(-(-n // page) for n in lens) * 4
        if case["op"] == "decode":
            return {"bytes": sum(lens) * row + io, "flops": 4 * sum(lens) * hq * dim}
        seen = sum(min(n, case["n_sel"] * page) for n in lens)
        pages = sum(-(-n // page) for n in lens)
        return {"bytes": seen * row + pages * hkv * dim * 4 + io + b * hkv * case["n_sel"] * 4,
                "flops": 4 * seen * hq * dim + 4 * pages * hq * dim}
    if case["op"] == "append":
        n = case["rows"]
        size = 4 if case["dtype"] == "float32" else 2
        # rows read, codes written, codes read again and values written by the gather
        return {"bytes": n * hkv * dim * 2 * (size + 2) + 2 * n * row + -(-n // page) * hkv * dim * 4,
                "flops": n * hkv * dim * (12 if case["rope"] else 9)}
    if case["op"] == "reorder":
        pages = b * -(-3 * case["ctx"] // 4 // page)
        copies = max(0, b // 2 - b // 10)
        return {"bytes": 2 * copies * case["layers"] * page_bytes + 16 * pages, "flops": 4 * pages}
    n = case["pages"]
    live = max(1, 6 * n // 10)
    return {"bytes": 2 * (live * (n - live) // n) * case["layers"] * page_bytes + 16 * n, "flops": 4 * n}


# ---------------------------------------------------------------- the definition in 64 bits

def _places():
    """For K and V, each token's and dim's byte in a cell and its shift, by the layout's words."""
    at = torch.zeros(2, 16, 64, dtype=torch.long)
    shift = torch.zeros(2, 16, 64, dtype=torch.long)
    meta = torch.zeros(2, 16, dtype=torch.long)
    for t in range(16):
        for d in range(64):
            at[0, t, d] = (t % 8) * 64 + (d // 16) * 16 + (t // 8) * 8 + d % 16 // 2
            at[1, t, d] = (512 + (d // 8) * 64 + (t % 8 // 2) * 16 + (t // 8) * 8 + (d % 8 // 4) * 4 + (t % 2) * 2
                           + d % 4 // 2)
            shift[:, t, d] = 4 * (d % 2)
        meta[0, t] = 1024 + (t % 8) * 8 + (t // 8) * 4
        meta[1, t] = 1088 + (t % 8) * 8 + (t // 8) * 4
    return at.cuda(), shift.cuda(), meta.cuda()


def _bf16_bits(lo, hi):
    """Two bytes as the bf16 number they are, in 64 bits."""
    return ((lo.int() << 16) | (hi.int() << 24)).view(torch.float32).double()


def _read(cells, which, places):
    at, shift, meta = (x[which] for x in places)
    code = (cells[..., at.reshape(-1)].int() >> shift.reshape(-1)) & 15
    d = _bf16_bits(cells[..., meta], cells[..., meta + 1])
    m = _bf16_bits(cells[..., meta + 2], cells[..., meta + 3])
    return code.reshape(*cells.shape[:-1], 16, 64).double() * d[..., None] + m[..., None]


def _rotate(x, pos, theta):
    """One vector [..., dim] at one position, by complex numbers."""
    dim = x.shape[-1]
    turn = torch.tensor([pos * math.pow(theta, -2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64,
                        device=x.device)
    z = torch.complex(x[..., :dim // 2].double(), x[..., dim // 2:].double()) * torch.polar(torch.ones_like(turn), turn)
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    places = _places()
    if case["op"] in ("decode", "sparse"):
        return _exact_decode(s, case, places)
    if case["op"] == "append":
        return _exact_append(s, case)
    # pages move as they are: whole numbers, but for the summaries, which are copies
    return None


def _exact_decode(s, case, places):
    b, hq, hkv, dim, page = (case[x] for x in ("batch", "hq", "hkv", "dim", "page"))
    grp = hq // hkv
    out = torch.zeros(b, hq, dim, dtype=torch.float64, device="cuda")
    for i in range(b):
        pos = int(s["pos"][i])
        n = pos // page + 1
        ids = s["table"][i, :n].long()
        q = _rotate(s["q"][i].reshape(hq, dim), pos, 10000.0).reshape(hkv, grp, dim)
        if case["op"] == "decode":
            lists = [list(range(n))] * hkv
        else:
            near = s["summary"][ids].double()  # [n, hkv, 2, dim]
            lists = []
            for h in range(hkv):
                lo, hi = near[:, h, 0], near[:, h, 1]
                bound = torch.stack([torch.maximum(x * lo, x * hi).sum(-1) for x in q[h]]).amax(0).tolist()
                order = sorted(range(n), key=lambda p: (p != n - 1, -bound[p], p))
                lists.append(sorted(order[:case["n_sel"]]))
        cells = s["pool"][ids].reshape(n, hkv, page // 16, dim // 64, CELL)
        for h in range(hkv):
            pick = torch.tensor(lists[h], device="cuda")
            tokens = (pick[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
            mine = cells[pick, h]
            k, v = (_read(mine, w, places).transpose(2, 3).reshape(-1, dim)[tokens <= pos] for w in (0, 1))
            p = torch.softmax(q[h] @ k.T / math.sqrt(dim), -1)
            out[i, h * grp:(h + 1) * grp] = p @ v
    out = out.reshape(b, hq * dim)
    return out if case["op"] == "decode" else dict(sel=None, out=out)


def _exact_append(s, case):
    hkv, dim, page, rows = (case[x] for x in ("hkv", "dim", "page", "rows"))
    cu = list(range(rows + 1)) if s["cu"] is None else s["cu"].tolist()
    summary = s["summary"].double()
    got = [torch.empty(rows, hkv * dim, dtype=torch.float64, device="cuda") for _ in range(2)]
    half = dim // 2
    rate = torch.tensor([math.pow(s["theta"] or 1.0, -2.0 * i / dim) for i in range(half)], dtype=torch.float64,
                        device="cuda")
    for i in range(case["batch"]):
        a, z, start = cu[i], cu[i + 1], int(s["pos"][i])
        k, v = (s[x][a:z].reshape(-1, hkv, dim).double() for x in ("k", "v"))
        if s["theta"] is not None:
            turn = torch.arange(start, start + z - a, dtype=torch.float64, device="cuda")[:, None] * rate
            w = torch.complex(k[..., :half], k[..., half:]) * torch.polar(torch.ones_like(turn), turn)[:, None]
            k = torch.cat([w.real, w.imag], -1)
        for x, to in zip((k, v), got):
            x = x.reshape(-1, 64)
            m = x.min(1).values.float().bfloat16().double()
            d = torch.clamp(((x.max(1).values - m) / 15).float().bfloat16().double(), min=D_MIN)
            steps = (torch.arange(15, device="cuda") + 0.5) * d[:, None]
            code = torch.searchsorted(steps, (x - m[:, None]).contiguous(), right=True)
            to[a:z] = (code * d[:, None] + m[:, None]).reshape(z - a, hkv * dim)
        kb = k.float().bfloat16().double()
        for p in range(start // page, (start + z - a - 1) // page + 1):
            lo, hi = max(start, p * page), min(start + z - a, (p + 1) * page)
            part = kb[lo - start:hi - start]
            at = int(s["table"][i, p])
            low, high = part.amin(0), part.amax(0)
            if lo > p * page:
                low, high = torch.minimum(low, summary[at, :, 0]), torch.maximum(high, summary[at, :, 1])
            summary[at, :, 0], summary[at, :, 1] = low, high
    return dict(k=got[0], v=got[1], summary=summary)
